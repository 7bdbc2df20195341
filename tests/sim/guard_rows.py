"""TEST INFRASTRUCTURE: the row operators on the CPU simulator with every operand, output and workspace ending (or beginning)
exactly at an inaccessible page; a read or write outside one faults.

    python tests/sim/guard_rows.py <norm|dropout|join> <end|begin>
"""
import faulthandler
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

SHAPES = [(1, 1), (5, 3), (3, 8), (4, 13), (2, 35), (3, 64), (2, 250), (2, 513), (2, 1030), (1, 2055), (1, 4099)]
LONG = (1, 8197)
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def main():
    faulthandler.enable()
    case, where = sys.argv[1:]
    from fiery_amd import native, row_ops
    from tests.sim.build_sim import build
    from tests.sim.guard_check import guarded
    lib = native.Lib(build())
    real_empty = torch.empty

    def empty(*shape, dtype=None, device=None, **kw):
        t = real_empty(*shape, dtype=dtype, device=device, **kw)
        return place(t) if t.numel() and t.device.type == 'cpu' else t

    def place(t):
        return guarded(t, where)

    def rows(shape, dtype):
        return place(torch.randn(*shape).to(dtype)).requires_grad_()

    torch.manual_seed(0)
    rng = place(row_ops.dropout_rng(4, 'cpu'))
    torch.empty = empty
    done = 0
    for shape in SHAPES + [LONG]:
        for dtype in TYPES if shape is not LONG else TYPES[1:2]:
            x, w, b = rows(shape, dtype), rows(shape[-1:], dtype), rows(shape[-1:], dtype)
            if case == 'norm':
                y = row_ops.layer_norm(x, w, b, lib=lib)
                torch.autograd.grad(y, (x, w, b), rows(shape, dtype).detach())
            for per in ('element', 'channel', 'sample') if shape[-1] < 1000 else ('element',):
                for stream in {dtype, torch.float32}:
                    r = rows(shape, stream)
                    if case == 'dropout':
                        y = row_ops.dropout(x, 0.4, rng, per=per, residual=r, lib=lib)
                        torch.autograd.grad(y, (x, r), rows(shape, stream).detach())
                        row_ops.dropout(x.detach(), 0.4, rng, per=per, lib=lib)
                    elif case == 'join':
                        y, h = row_ops.dropout_add_layer_norm(x, r, w, b, 0.4, rng, per=per, lib=lib)
                        torch.autograd.grad((y, h), (x, r, w, b), (rows(shape, dtype).detach(), rows(shape, stream).detach()))
            done += 1
    print(f'ok {case} {where} ({done} shapes)', flush=True)


if __name__ == '__main__':
    main()
