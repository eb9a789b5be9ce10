"""The largest calls: past 2^32 threads a launch (more rows than one launch takes), and what no launch takes."""
import pytest
import torch

from lira_amd import _lib

A = 4096  # an aligned address that is never read: every call below ends before a launch


@pytest.mark.parametrize("m,n,k", [(17, 1 << 33, 100), (4096, 1 << 31, 1000), ((1 << 31) - 1, 1 << 20, 64), (17, (1 << 31) + 129, 128)])
def test_products_of_more_tiles_than_a_launch_has_threads(m, n, k):
    lib = _lib.load()
    assert lib.lira_mx4_matmul(A, A, m, m, A, A, n, n, k, 1.0, None, 0, A, 1, n, None) == -6
    assert "too many tiles" in lib.lira_last_error().decode()
    # (and before rows are packed into the workspace)
    assert lib.lira_mx4_linear(A, 0, m, k, k, A, A, n, n, 1.0, None, 0, A, 1, n, A, 1 << 60, None) == -6
    assert "too many tiles" in lib.lira_last_error().decode()


@pytest.mark.parametrize("t,ok", [(1e-20, False), (1e-19, False), (1.1e-19, True), (1.8e19, True), (1.9e19, False), (1e30, False)])
def test_temperatures_whose_square_leaves_fp32(t, ok):
    """The loss has the factor T^2: past fp32's end it was NaN or infinite, and 0 below its smallest number."""
    lib = _lib.load()
    rc = lib.lira_distill_topk(A, 0, 0, 100, 100, A, 32, A, 5, t, None, A, None, None, 0, None, 0, None, 0, None)  # (of no rows)
    assert (rc == 0) if ok else (rc == -1 and "square" in lib.lira_last_error().decode())


@pytest.mark.gpu
def test_more_packed_rows_than_a_launch_takes():
    """2^28 rows by workgroups of 16 and 2^27 by workgroups of 8 are 2^32 threads."""
    from lira_amd import mx4_quantize
    n = (1 << 28) + 21
    values = torch.tensor([0, 1, -1.5, 2, 3, -0.5, 6], device="cuda")  # (a power of two times an element: exact)
    x = values[torch.arange(n, device="cuda") % 7].bfloat16()[:, None]
    t = mx4_quantize(x)
    assert torch.equal(t.dequantize(torch.bfloat16), x)
    assert torch.equal(t.dequantize(torch.float32), x.float())
    at = (1 << 28) - 16  # (the first row of the second launch)
    for lo in (0, at - 20, n - 40):
        part = mx4_quantize(x[lo:lo + 40])
        assert torch.equal(t.codes[:, lo:lo + 40], part.codes) and torch.equal(t.scales[:, lo:lo + 40], part.scales)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,top", [((1 << 26) + 9, 8, 1), ((1 << 24) + 9, 72, 65)])
def test_more_distilled_rows_than_a_launch_takes(rows, vocab, top):
    """A wave a row, and a workgroup a row where the entries are more than 64: bit for bit as in two halves."""
    from lira_amd import distill_topk_loss, distill_topk_loss_and_grad
    g = torch.Generator(device="cuda").manual_seed(top)
    z = torch.randn(rows, vocab, generator=g, device="cuda")
    ti = torch.randint(-1, vocab, (rows, top), generator=g, device="cuda", dtype=torch.int32)
    tv, w, lse = (torch.randn(*s, generator=g, device="cuda") for s in ((rows, top), (rows,), (rows,)))
    loss, dz = distill_topk_loss_and_grad(z, ti, tv, 2.0, lse, w)
    half = rows // 2
    for s in (slice(0, half), slice(half, rows)):
        a, b = distill_topk_loss_and_grad(z[s], ti[s], tv[s], 2.0, lse[s], w[s])
        assert torch.equal(loss[s], a) and torch.equal(dz[s], b)
        del a, b
    z.requires_grad_(True)
    got = distill_topk_loss(z, ti, tv, 2.0, lse, reduction="none")
    (d2,) = torch.autograd.grad(got, z, w)
    del dz, loss
    for s in (slice(0, half), slice(half, rows)):
        part = z[s].detach().requires_grad_(True)
        a = distill_topk_loss(part, ti[s], tv[s], 2.0, lse[s], reduction="none")
        (d,) = torch.autograd.grad(a, part, w[s])
        assert torch.equal(got[s], a) and torch.equal(d2[s], d)
        del part, a, d
