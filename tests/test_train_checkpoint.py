"""Dropout of the training graph under activation checkpointing: the forward pass that is run again draws the masks of the first."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from fiery_amd import row_ops
from fiery_amd import train_graph as tg
from tests.test_row_ops import on  # noqa: F401  (the two backends)
from tests.test_train_dropout import _MBConv, _block, _mask


def _same(t):
    return t


def _bottleneck(on):  # noqa: F811
    blk, x = _block(on)
    blk.layers.dropout.p = 0.5
    graph = tg.TrainGraph(None, on.lib)
    return graph, (lambda t: graph.bottleneck(t, blk)), x, list(blk.parameters())


def _pass(on):  # noqa: F811
    first, x = _block(on)
    second, _ = _block(on, True)
    first.layers.dropout.p, second.layers.dropout.p = 0.5, 0.3
    graph = tg.TrainGraph(None, on.lib)

    @tg._counts_batches_once
    def entry(self, t):
        return self.bottleneck(self.bottleneck(t, first), second)
    return graph, (lambda t: entry(graph, t)), x, list(first.parameters()) + list(second.parameters())


def _drop_connect(on):  # noqa: F811
    torch.manual_seed(5)
    blk = _MBConv().block.train().to(on.device)
    graph = tg.TrainGraph(None, on.lib)
    return graph, (lambda t: graph._mbconv(blk, t, 0.5)), torch.randn(5, 8, 6, 7).to(on.device), [p for p in blk.parameters() if p.requires_grad]


CASES = {'bottleneck': _bottleneck, 'pass': _pass, 'drop_connect': _drop_connect}


@pytest.mark.parametrize('case', list(CASES))
def test_checkpointed_gradients_are_those_of_the_plain_pass(on, case, monkeypatch):  # noqa: F811
    """The same draws of torch's generator, once plainly and once through checkpoint: outputs equal, gradients equal to the rounding of
    sums of another order (1e-5 of the largest value, as the suite's other block tests).  Another mask is a difference of order one."""
    monkeypatch.setattr(tg, 'DROP_CONNECT', 'counter')
    graph, f, x, params = CASES[case](on)
    graph.dropout_rng = row_ops.dropout_rng(17, on.device)
    leaf = x.clone().requires_grad_()
    torch.manual_seed(40)
    with torch.autograd.graph.saved_tensors_hooks(_same, _same):
        want = f(leaf)
    gy = torch.randn(want.shape, generator=torch.Generator().manual_seed(1)).to(on.device)
    want_grads = torch.autograd.grad(want, [leaf] + params, gy, allow_unused=True)
    torch.manual_seed(40)
    got = checkpoint(f, leaf, use_reentrant=False)
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()
    graph.dropout_rng[1] += 5                                      # whatever becomes of the counter meanwhile
    f(x)
    got_grads = torch.autograd.grad(got, [leaf] + params, gy, allow_unused=True)
    assert any(g is not None for g in got_grads[1:])
    for a, b in zip(got_grads, want_grads):
        assert (a is None) == (b is None)
        if a is not None:
            assert (a - b).abs().max() <= 1e-5 * max(1.0, b.abs().max())
    assert not torch.equal(checkpoint(f, leaf, use_reentrant=False), got)       # the next pass draws others


def test_checkpointed_masks_are_numbered_by_torchs_generator(on):  # noqa: F811
    """Inside a checkpoint the call number is drawn on the CPU, whose state checkpoint restores, under the model's seed; the counter that
    numbers the other passes stays."""
    graph = tg.TrainGraph(None, on.lib)
    graph.dropout_rng = row_ops.dropout_rng(23, on.device)
    graph.dropout_rng[1] += 9
    x = torch.ones(3, 8, 4, 5, device=on.device, requires_grad=True)
    torch.manual_seed(41)
    y = checkpoint(lambda t: graph.dropout_add(t, torch.zeros_like(t), 0.5, 'channel'), x, use_reentrant=False)
    torch.manual_seed(41)
    number = int(torch.randint(1 << 62, (1,)))
    m = _mask(on, x.shape, 0.5, 23, number, 'channel')
    assert torch.equal(y, m)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], m)
    assert graph.dropout_rng.tolist() == [23, 9]
    plain = graph.dropout_add(x, torch.zeros_like(x), 0.5, 'channel')
    assert torch.equal(plain, _mask(on, x.shape, 0.5, 23, 9, 'channel')) and graph.dropout_rng.tolist() == [23, 10]


def test_reentrant_checkpoints_are_refused(on):  # noqa: F811
    """Their first pass looks like any other; the second one, inside the backward pass, is an error and not a gradient of other masks."""
    graph, f, x, _ = _bottleneck(on)
    y = checkpoint(f, x.clone().requires_grad_(), use_reentrant=True)
    with pytest.raises(RuntimeError, match='use_reentrant=False'):
        y.sum().backward()
    assert f(x).shape == y.shape                                   # the next pass works


def test_a_captured_checkpoint_is_refused(sim, monkeypatch):
    """Its number would be part of the capture: every replay would draw the same masks."""
    graph = tg.TrainGraph(None, sim)
    x = torch.ones(2, 8, 3, 3, requires_grad=True)
    graph.dropout_add(x, x, 0.5, 'channel')
    monkeypatch.setattr(tg, '_capturing', lambda t: True)
    with pytest.raises(RuntimeError, match='captured'):
        checkpoint(lambda t: graph.dropout_add(t, t, 0.5, 'channel'), x, use_reentrant=False, preserve_rng_state=False)
    graph.dropout_add(x, x, 0.5, 'channel')
