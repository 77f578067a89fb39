"""Workspace sizes of the model operators: one that holds a batch holds every smaller one. No GPU is needed."""
import ctypes as C

import pytest

from tierstream_amd import ops

AT = [1, 2, 255, 256, 1000, 2047, 2048, 2049, 4096, 4097, 16383, 16384, 16385, 65536, 131071, 131072, 131073, 132000, 135168, 196608,
      196609, 200000, 262144, 262145, 1 << 20, (1 << 20) + 1, (1 << 21) - 1]


@pytest.mark.parametrize("n,d,f", [(512, 64, 72), (512, 256, 512), (7, 33, 47), (1, 4096, 1024), (128, 32, 64)])
@pytest.mark.parametrize("top_k", [1, 2, 8])
@pytest.mark.parametrize("kind", [ops.BF16, ops.F16, ops.Q4])
def test_block_sizes_grow_with_rows(n, d, f, top_k, kind):
    if kind == ops.Q4 and (d % 32 or f % 32):
        d, f = 64, 96
    e = ops.TsaExperts(n_experts=n, d_model=d, d_ff=f, w_type=kind)
    rows = sorted({r // k for r in AT for k in (1, top_k) if r // k} | {r // top_k + 1 for r in AT if (r // top_k + 1) * top_k < 1 << 24})
    sizes = [ops._ops().tsa_ffn_workspace(C.byref(e), r, top_k) for r in rows]
    assert min(sizes) > 0 and sizes == sorted(sizes)
    if kind != ops.Q4:
        sizes = [ops._ops().tsa_ffn_backward_workspace(C.byref(e), r, top_k) for r in rows]
        assert min(sizes) > 0 and sizes == sorted(sizes)


@pytest.mark.parametrize("n_in,n_out", [(7168, 256), (4096, 28672), (2048, 7168), (64, 16), (96, 40000), (8192, 513)])
@pytest.mark.parametrize("kind", [ops.BF16, ops.Q4])
@pytest.mark.parametrize("x", [16, 18])
def test_product_sizes_grow_with_rows(n_in, n_out, kind, x):
    """For one and the same alignment of x and the weights."""
    sizes = []
    for rows in [*range(1, 140), *AT]:
        if rows * n_out < 1 << 37:
            a = ops.TsaLinearArgs(x=x, x_stride=n_in, w=16, w_stride=n_in, rows=rows, n_in=n_in, n_out=n_out, x_type=ops.BF16, w_type=kind,
                                  y_type=ops.BF16)
            sizes.append((rows, ops._ops().tsa_linear_workspace(C.byref(a))))
    sizes = [s for _, s in sorted(sizes)]
    assert sizes == sorted(sizes) and (x == 16) == (sizes[-1] == 0)
