"""TEST INFRASTRUCTURE: the joined row operator's gradient at the unrounded h on the CPU simulator, every operand, output and
workspace ending (or beginning) exactly at an inaccessible page; a read or write outside one faults.

    python tests/sim/guard_unrounded.py <end|begin>
"""
import faulthandler
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)


def main():
    faulthandler.enable()
    where = sys.argv[1]
    from fiery_amd import native
    from tests.sim.build_sim import build
    from tests.sim.guard_check import guarded
    from tests.sim.guard_rows import SHAPES
    lib = native.Lib(build())
    torch.manual_seed(0)
    rng = guarded(torch.tensor([4, 5]), where)
    keep, done = [], 0

    def given(shape, dtype):
        keep.append(guarded(torch.randn(*shape).to(dtype), where))
        return keep[-1].data_ptr()
    for rows, c in SHAPES:
        n = lib.dll.fiery_layer_norm_bwd_workspace_floats(rows, c)
        for dtype in (torch.bfloat16, torch.float16)[:1 if c > 1000 else 2]:
            t = native.ROW_TYPES[dtype]
            x, par = lambda: given((rows, c), dtype), lambda: given((c,), dtype)
            stats, used = guarded(torch.rand(2 * rows) + 0.5, where), guarded(torch.zeros(2, dtype=torch.int64), where)
            mean, rstd = stats.data_ptr(), stats.data_ptr() + 4 * rows
            ws = given((n,), torch.float32) if n else None
            for threshold, share, one in ((20000, 1, 0), (20000, 2, 1), (0, 1, 0))[:1 if c > 8000 else 3]:
                lib.check(lib.dll.fiery_dropout_add_layer_norm_fwd_unrounded(x(), c, t, x(), c, t, rows, c, par(), par(), t, 1e-5, threshold, rng.data_ptr(), 1, share,
                                                                             one, used.data_ptr(), x(), c, x(), c, mean, rstd, None))
                for dh in (None, x())[1 if c > 8000 else 0:]:
                    lib.check(lib.dll.fiery_dropout_add_layer_norm_bwd_unrounded(x(), c, dh, c, x(), c, x(), c, t, rows, c, par(), t, mean, rstd, threshold,
                                                                                 used.data_ptr(), share, one, x(), c, x(), c, par(), par(), ws, n, None))
            done += 1
            keep.clear()
    print(f'ok unrounded {where} ({done} shapes)', flush=True)


if __name__ == '__main__':
    main()
