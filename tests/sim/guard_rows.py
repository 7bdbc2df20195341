"""TEST INFRASTRUCTURE: the row operators' entry points on the CPU simulator with every operand, output and workspace ending (or
beginning) exactly at an inaccessible page; a read or write outside one faults.

    python tests/sim/guard_rows.py <norm|dropout|join> <end|begin>
"""
import faulthandler
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

SHAPES = [(1, 1), (5, 3), (3, 8), (4, 13), (2, 35), (3, 64), (2, 250), (2, 513), (2, 1030), (1, 2055), (1, 4099), (90, 24), (1, 8197)]
TYPES = (torch.float32, torch.bfloat16, torch.float16)
F32 = torch.float32


def main():
    faulthandler.enable()
    case, where = sys.argv[1:]
    from fiery_amd import native
    from tests.sim.build_sim import build
    from tests.sim.guard_check import guarded
    lib = native.Lib(build())
    torch.manual_seed(0)
    kind = native.ROW_TYPES
    rng = guarded(torch.tensor([4, 5]), where)

    def given(shape, dtype):
        t = guarded(torch.randn(*shape).to(dtype), where)
        keep.append(t)
        return t.data_ptr()

    def room(shape, dtype):
        return given(shape, dtype)
    done, keep = 0, []
    for rows, c in SHAPES:
        long = c > 1000
        n = lib.dll.fiery_layer_norm_bwd_workspace_floats(rows, c)
        for dtype in TYPES[1:2] if c > 8000 else TYPES:
            t = kind[dtype]
            x = lambda d=dtype: given((rows, c), d)
            par = lambda: given((c,), dtype)
            stats = guarded(torch.rand(2 * rows) + 0.5, where)
            mean, rstd = stats.data_ptr(), stats.data_ptr() + 4 * rows
            ws = given((n,), F32) if n else None
            if case == 'norm':
                lib.check(lib.dll.fiery_layer_norm_fwd(x(), c, t, rows, c, par(), par(), t, 1e-5, room((rows, c), dtype), c, mean, rstd, None))
                lib.check(lib.dll.fiery_layer_norm_bwd(x(), c, x(), c, t, rows, c, par(), t, mean, rstd, room((rows, c), dtype), c, par(), par(), ws, n, None))
            for share, one in ((1, 0), (2, 0), (2, 1)) if not long else ((1, 0),):
                for stream in {dtype, F32}:
                    s, used = kind[stream], guarded(torch.zeros(2, dtype=torch.int64), where)
                    if case == 'dropout':
                        for res in (None, x(stream)):
                            lib.check(lib.dll.fiery_dropout(x(), c, t, res, c, rows, c, 20000, rng.data_ptr(), 1, share, one, used.data_ptr(),
                                                            room((rows, c), stream), c, s, None))
                        lib.check(lib.dll.fiery_dropout(x(stream), c, s, None, 0, rows, c, 20000, used.data_ptr(), 0, share, one, None,
                                                        room((rows, c), dtype), c, t, None))
                    elif case == 'join':
                        lib.check(lib.dll.fiery_dropout_add_layer_norm_fwd(x(), c, t, x(stream), c, s, rows, c, par(), par(), t, 1e-5, 20000, rng.data_ptr(), 1,
                                                                           share, one, used.data_ptr(), room((rows, c), dtype), c, room((rows, c), stream), c,
                                                                           mean, rstd, None))
                        for dh in (None, x(stream)):
                            lib.check(lib.dll.fiery_dropout_add_layer_norm_bwd(x(), c, dh, c, x(stream), c, t, s, rows, c, par(), t, mean, rstd, 20000,
                                                                               used.data_ptr(), share, one, room((rows, c), dtype), c,
                                                                               room((rows, c), stream), c, par(), par(), ws, n, None))
            done += 1
            keep.clear()
    print(f'ok {case} {where} ({done} shapes)', flush=True)


if __name__ == '__main__':
    main()
