"""C as a column slice of a wider matrix with 16-byte aligned rows and an N that is no multiple of 8: the columns behind
the slice stay as they were (a TMA store writes whole 16-byte pieces, so these shapes go by ordinary stores)."""
import pytest

from helpers import assert_parity, make_inputs, to_device, to_host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("force", [0, 1, 2, 3, 4, 5, 6, 10, 12])
@pytest.mark.parametrize("n,ldc", [(57, 64), (251, 256), (1027, 1032)])
def test_columns_behind_an_odd_slice_stay(ctx, oracle, force, n, ldc):
    import torch
    m, k = 300, 128
    a, b = make_inputs(oracle, m, n, k, 91)
    buf = torch.full((m, ldc), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.set("force_kernel", force)
    try:
        ctx.gemm(to_device(a), to_device(b), out=buf[:, :n])
        ctx.poll()
    finally:
        ctx.set("force_kernel", 0)
    assert (buf[:, n:] == 7).all()
    assert_parity(oracle, to_host(buf[:, :n].contiguous()), oracle.gemm_bf16(a, b), k, oracle.max_abs_bf16(a),
                  oracle.max_abs_bf16(b), f"n {n}, ldc {ldc}, kernel {force}")
