"""Dropout inside the training graph: the Bottleneck's Dropout2d and the trunk's drop-connect on the library's counter-based
dropout, on the simulated kernels and the GPU."""
import pytest
import torch

from fiery_amd import row_ops
from fiery_amd import train_graph as tg
from fiery_amd.modules import ResidualBottleneck
from tests.test_row_ops import kept, on  # noqa: F401  (the two backends)


def _block(on, downsample=False, cin=16, cout=16):
    torch.manual_seed(3)
    blk = ResidualBottleneck(cin, cout, downsample=downsample).train()
    return blk.to(on.device), torch.randn(3, cin, 6, 8).to(on.device)


def _mask(on, shape, p, seed, call, per):
    n, c, h, w = shape
    return kept((n, h * w, c), p, seed, call, per).view(n, h, w, c).permute(0, 3, 1, 2).float().to(on.device)


@pytest.mark.parametrize('downsample,cout', [(False, 16), (True, 16), (False, 24)])
def test_bottleneck_drops_channels_of_its_branch(on, downsample, cout):  # noqa: F811
    """`layers.dropout.p` > 0: whole channels of the branch, scaled, before the skip is added; gradients through the same mask.
    p = 0 and eval() give what they gave before.  The sums and products of the two sides differ in 32-bit rounding only: 1e-5 of
    the largest value covers the 3 x 3 convolutions' different orders as elsewhere in the suite."""
    blk, x = _block(on, downsample, 16, cout)
    p, seed = 0.4, 1234567
    graph = tg.TrainGraph(None, on.lib)
    captured = {}
    plain_add = lambda r, skip, p, per: captured.update(r=r, skip=skip) or r + skip
    graph.dropout_add = plain_add
    blk.layers.dropout.p = p
    leaf = x.clone().requires_grad_()
    graph.bottleneck(leaf, blk)
    r, skip = captured['r'], captured['skip']
    m = _mask(on, r.shape, p, seed, 0, 'channel')
    want = r * m + skip
    gy = torch.randn(want.shape, generator=torch.Generator().manual_seed(1)).to(on.device)
    params = [q for q in blk.parameters() if q.requires_grad]
    want_grads = torch.autograd.grad(want, [leaf] + params, gy)

    graph = tg.TrainGraph(None, on.lib)
    graph.dropout_rng = row_ops.dropout_rng(seed, on.device)
    leaf2 = x.clone().requires_grad_()
    got = graph.bottleneck(leaf2, blk)
    assert graph.dropout_rng.tolist() == [seed, 1]                   # a block on its own advances the numbers at once
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()
    for a, b in zip(torch.autograd.grad(got, [leaf2] + params, gy), want_grads):
        assert (a - b).abs().max() <= 1e-5 * max(1.0, b.abs().max())
    again = graph.bottleneck(x, blk)
    assert not torch.equal(again, got)                               # the next call's masks are others
    blk.layers.dropout.p = 0.0
    off = graph.bottleneck(x, blk)
    assert graph.dropout_rng.tolist() == [seed, 2]
    blk.layers.dropout.p = p
    blk.layers.dropout.eval()
    assert torch.equal(graph.bottleneck(x, blk), off)


class _MBConv(torch.nn.Module):
    def __init__(self):
        super().__init__()
        from fiery_amd.backbone import MBConvBlock
        self.block = MBConvBlock(3, 1, 1, 8, 8, 16)


def test_drop_connect_by_counter(on, monkeypatch):  # noqa: F811
    torch.manual_seed(5)
    blk = _MBConv().block.train().to(on.device)
    x = torch.randn(5, 8, 6, 7).to(on.device)
    graph = tg.TrainGraph(None, on.lib)
    graph.dropout_rng = row_ops.dropout_rng(99, on.device)
    plain = graph._mbconv(blk, x, 0.0)
    monkeypatch.setattr(tg, 'DROP_CONNECT', 'counter')
    got = graph._mbconv(blk, x, 0.5)
    m = _mask(on, x.shape, 0.5, 99, 0, 'sample')
    assert 0 < int((m[:, 0, 0, 0] == 0).sum()) < 5
    want = (plain - x) * m + x
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()
    assert torch.equal(got[m[:, 0, 0, 0] == 0], x[m[:, 0, 0, 0] == 0])
    # the default draws from torch's generator as before and leaves the counter alone
    monkeypatch.setattr(tg, 'DROP_CONNECT', 'torch')
    numbers = graph.dropout_rng.tolist()
    torch.manual_seed(11)
    one = graph._mbconv(blk, x, 0.5)
    torch.manual_seed(11)
    keep = torch.floor(0.5 + torch.rand(5, 1, 1, 1, device=on.device))
    assert (one - ((plain - x) / 0.5 * keep + x)).abs().max() <= 1e-5 * want.abs().max()
    assert graph.dropout_rng.tolist() == numbers


def test_a_pass_numbers_its_dropouts_and_advances_once(sim):
    """Inside an entry point every dropout has its own number; the tensor moves on when the pass ends, also when it fails."""
    graph = tg.TrainGraph(None, sim)
    graph.dropout_rng = row_ops.dropout_rng(7, 'cpu')
    x = torch.ones(2, 8, 3, 3)
    zero = torch.zeros_like(x)

    @tg._counts_batches_once
    def two(self, fail=False):
        out = [self.dropout_add(x, zero, 0.5, 'channel') for _ in range(2)]
        assert self.dropout_rng.tolist()[1] % 2 == 0
        if fail:
            raise KeyError('x')
        return out
    a, b = two(graph)
    assert graph.dropout_rng.tolist() == [7, 2]
    assert torch.equal(a, _mask(type('D', (), dict(device='cpu')), x.shape, 0.5, 7, 0, 'channel') * x)
    assert torch.equal(b, _mask(type('D', (), dict(device='cpu')), x.shape, 0.5, 7, 1, 'channel') * x)
    with pytest.raises(KeyError):
        two(graph, fail=True)
    assert graph.dropout_rng.tolist() == [7, 4]


def test_model_keeps_its_numbers_and_its_checkpoint(sim):
    """The numbers live on the model between passes and not in its state_dict; without a seed of its own the model takes one from
    torch's."""
    import types
    model = types.SimpleNamespace()
    first = tg.TrainGraph(None, sim)
    first.m = model
    x = torch.ones(1, 8, 2, 2)
    torch.manual_seed(21)
    y = first.dropout_add(x, torch.zeros_like(x), 0.5, 'channel')
    seed, call = model.dropout_rng.tolist()
    assert call == 1
    second = tg.TrainGraph(None, sim)
    second.m = model
    second.dropout_add(x, torch.zeros_like(x), 0.5, 'channel')
    assert model.dropout_rng.tolist() == [seed, 2]
    torch.manual_seed(21)
    third = tg.TrainGraph(None, sim)
    third.m = types.SimpleNamespace()
    assert torch.equal(third.dropout_add(x, torch.zeros_like(x), 0.5, 'channel'), y)


@pytest.mark.gpu
def test_a_models_training_pass_with_dropout(hip):
    """p > 0 in every Bottleneck of the tiny model: one number per block and pass, finite gradients everywhere, the same outputs from
    the same numbers (to the rounding of the pooling's atomics: 2e-4 of the largest value, as the suite's other training passes), others
    from the next."""
    from fiery_amd.model import Fiery
    from tests.golden.make_golden import training_loss, training_model_case
    from tests.helpers import forward_case, randomise_weights
    cfg, B, n_cam = training_model_case()
    torch.manual_seed(0)
    model = Fiery(cfg)
    randomise_weights(model)
    keys = list(model.state_dict())
    model = model.cuda().train()
    blocks = [m for m in model.modules() if isinstance(m, ResidualBottleneck)]
    for b in blocks:
        b.layers.dropout.p = 0.1
    lifted, K, E, ego, labels, noise = forward_case(cfg, model.receptive_field, model.n_future, model.depth_channels, model.bev_size, B, n_cam,
                                                    with_labels=True, with_noise=True)
    args = [t.cuda() for t in (lifted, K, E, ego, labels, noise)]

    def run(call):
        model.dropout_rng = row_ops.dropout_rng(77)
        model.dropout_rng[1] = call
        with torch.no_grad():
            for m in model.modules():                                # the running averages do not enter a pass in train() mode
                if isinstance(m, torch.nn.modules.batchnorm._BatchNorm):
                    m.reset_running_stats()
        return model.bev_forward(*args)
    out = run(0)
    assert model.dropout_rng.tolist() == [77, len(blocks)] and len(blocks) > 8
    training_loss(out).backward()
    grads = [p.grad for n, p in model.named_parameters() if not n.startswith('encoder.') and p.grad is not None]
    assert len(grads) > 100 and all(torch.isfinite(g).all() for g in grads)
    same, other = run(0), run(len(blocks))
    a, b, c = (o['instance_offset'].detach() for o in (out, same, other))
    scale = a.abs().max()
    assert (a - b).abs().max() <= 2e-4 * max(1.0, scale)
    assert (a - c).abs().max() > 1e-2 * scale
    assert list(model.state_dict()) == keys
