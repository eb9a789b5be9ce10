"""GPU: distillation from a teacher's top outputs against 64-bit references and differences."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
INF = float("inf")


def make(rows, vocab, top, dtype="fp32", ids=torch.int64, seed=0, masked=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (2 * torch.randn(rows, vocab, generator=g, device="cuda")).to(DT[dtype])
    tv, ti = torch.topk(z.float() + 1.5 * torch.randn(rows, vocab, generator=g, device="cuda"), top, dim=1)
    if masked:
        hide = torch.rand(rows, vocab, generator=g, device="cuda") < 0.3
        z.masked_fill_(hide.scatter_(1, ti, False), -INF)
        n = torch.randint(0, top + 1, (rows, 1), generator=g, device="cuda")
        ti = ti.masked_fill(torch.arange(top, device="cuda") >= n, -1)
    w = torch.randn(rows, generator=g, device="cuda")
    return z, ti.to(ids), tv, w


def ref(z, ti, tv, t, lse=None):
    """(loss, gradient of each row's loss, tolerances of both before the output's rounding) in 64 bits.

    fp32 arithmetic, eps = 2^-24: an exponent x of size up to R = max |z / T - max| is off by 2 (R + 1) eps
    (its scaling and subtraction round), which is the relative error of its exp; a sum of V terms in any
    order of chains of V / 64 adds loses (V / 64 + 8) eps.  So lse and every log q are off by
    D = (4 R + V / 64 + 16) eps + 2 |lse| eps, p and log p likewise with the teacher's range, and the
    hardware's exp and log add 4 eps each."""
    eps = 2.0 ** -24
    x = z.double() / t
    used = ti >= 0
    at = ti.long().clamp(min=0)
    logq = torch.log_softmax(x, 1)
    y = (tv.double() / t).masked_fill(~used, -INF)
    some = (y > -INF).any(1, keepdim=True)
    L = torch.logsumexp(y.masked_fill(~some, 0), 1, keepdim=True) if lse is None else lse.double()[:, None]
    logp = (y - L).masked_fill(y == -INF, -INF)
    p = logp.exp()
    s = p.sum(1, keepdim=True)
    lq = logq.gather(1, at)
    loss = t * t * torch.where(p > 0, p * (logp - lq), 0.0).sum(1)
    grad = (logq.exp().nan_to_num(nan=0.0) * s).scatter_add(1, at, -p) * t
    fin = x.masked_fill(x == -INF, 0)
    R = fin.abs().amax() * 2
    Rt = y.masked_fill(y == -INF, 0).abs().amax() * 2 + L.abs().amax()
    V = z.shape[1]
    D = (8 * R + 8 * Rt + V / 64 + 32) * eps
    tl = t * t * (torch.where(p > 0, p * (logp.abs() + lq.abs() + 1), 0.0).sum(1) * (D + 16 * eps) + s[:, 0] * D) + 1e-37
    tg = t * (logq.exp().nan_to_num(nan=0.0) * s).scatter_add(1, at, p) * (2 * D + 16 * eps) + 1e-37
    return loss, grad, tl, tg


def check_loss(got, want, tol):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def check_grad(got, want, tol):
    f = torch.finfo(got.dtype)
    tol = tol + f.eps / 2 * (want.abs() + tol) + f.smallest_normal * f.eps
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


CASES = [(1, 1, 1), (1, 7, 7), (3, 64, 5), (5, 257, 8), (64, 1000, 32), (17, 1024, 64), (2, 4097, 100), (33, 8192, 16),
         (4, 32768, 64), (3, 50001, 10), (2, 131072, 64), (1, 300000, 1024), (700, 40, 3), (600, 7, 2), (520, 2000, 64), (515, 16391, 65), (513, 70001, 12), (513, 140000, 20)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,vocab,top", CASES)
def test_loss_and_gradient(rows, vocab, top, masked, dtype):
    from lira_amd import distill_topk_loss, distill_topk_loss_and_grad
    for t, ids in ((1.0, torch.int32), (3.0, torch.int64)):
        z, ti, tv, w = make(rows, vocab, top, dtype, ids, rows + vocab, masked)
        loss, grad, tl, tg = ref(z, ti, tv, t)
        got, dz = distill_topk_loss_and_grad(z, ti, tv, t, row_weight=w)
        check_loss(got, loss, tl)
        check_grad(dz, grad * w.double()[:, None], tg * w.double().abs()[:, None] * 1.001)
        z.requires_grad_(True)
        got = distill_topk_loss(z, ti, tv, t, reduction="none")
        check_loss(got, loss, tl)
        (dz,) = torch.autograd.grad(got, z, w)
        check_grad(dz, grad * w.double()[:, None], tg * w.double().abs()[:, None] * 1.001)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reductions(reduction):
    from lira_amd import distill_topk_loss
    z, ti, tv, _ = make(3000, 130, 6, masked=True)
    ti[::3] = -1
    loss, grad, tl, tg = ref(z, ti, tv, 2.0)
    n = int((ti >= 0).any(1).sum()) if reduction == "mean" else 1
    z.requires_grad_(True)
    got = distill_topk_loss(z, ti, tv, 2.0, reduction=reduction)
    # (the reduction adds 3000 values, three a thread and then a tree: 32 roundings of the magnitudes' sum)
    assert abs(got.item() - float(loss.sum()) / n) <= float(tl.sum() + loss.abs().sum() * 32 * 2.0 ** -24) / n
    (3.0 * got).backward()
    check_grad(z.grad, 3.0 * grad / n, 3.01 * tg / n)
    assert not z.grad[::3].any()


def test_no_second_derivative():
    from lira_amd import distill_topk_loss
    z, ti, tv, _ = make(5, 70, 4)
    z.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(distill_topk_loss(z, ti, tv), z, create_graph=True)
    loss = distill_topk_loss(z, ti, tv)
    with torch.no_grad():
        z.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_saved_elsewhere():
    """The backward pass on what the hooks bring back (offloaded activations), not on the first addresses."""
    from lira_amd import distill_topk_loss
    z, ti, tv, w = make(40, 3000, 9, "bf16")
    z.requires_grad_(True)
    (want,) = torch.autograd.grad(distill_topk_loss(z, ti, tv, 2.0, reduction="none"), z, w)
    with torch.autograd.graph.save_on_cpu():
        loss = distill_topk_loss(z * 1.0, ti.clone(), tv.clone(), 2.0, reduction="none")
    junk = [torch.full_like(x, 7) for x in (z.detach(), ti, tv) for _ in range(4)]  # (over what was freed)
    (got,) = torch.autograd.grad(loss, z, w)
    assert torch.equal(got, want) and len(junk) == 12


def test_no_row_counts():
    from lira_amd import distill_topk_loss
    z, ti, tv, _ = make(5, 70, 4)
    z.requires_grad_(True)
    for ids, logits in ((torch.full_like(ti, -1), tv), (ti, torch.full_like(tv, -INF))):
        for red in ("mean", "sum", "none"):
            loss = distill_topk_loss(z, ids, logits, reduction=red)
            (g,) = torch.autograd.grad(loss.sum(), z)
            assert not loss.any() and not g.any()
    empty = torch.zeros(0, 70, device="cuda", requires_grad=True)
    loss = distill_topk_loss(empty, ti[:0], tv[:0])
    loss.backward()
    assert float(loss) == 0.0 and empty.grad.shape == (0, 70)


@pytest.mark.parametrize("vocab", [40, 9000])
def test_special_rows(vocab):
    """Masked students, entries of the same id, Inf and NaN, ids past the end."""
    from lira_amd import distill_topk_loss_and_grad
    z, ti, tv, _ = make(10, vocab, 6)
    z[0] = -INF                      # nothing left of the student
    z[1, ti[1, 2]] = -INF            # an entry names a masked output
    z[2, 3] = float("nan")
    z[3, 5] = INF
    ti[4, 1] = vocab                 # past the end
    tv[5, 0] = float("nan")
    ti[6, 1:4] = ti[6, 0]            # the same output four times
    tv[7, 1:] = -INF                 # one entry counts
    ti[8, :5] = -1
    loss, dz = distill_topk_loss_and_grad(z, ti, tv, 2.0)
    sane = [6, 7, 8, 9]  # (the rows with numbers alone: the tolerance goes by their range)
    want, _, tl, _ = ref(z[sane], ti[sane], tv[sane], 2.0)
    check_loss(loss[sane], want, tl)
    assert float(loss[0]) == INF and float(loss[1]) == INF
    for r in (2, 3, 4, 5):
        assert bool(torch.isnan(loss[r])) and bool(torch.isnan(dz[r]).all())
    sane = [1, 6, 7, 8, 9]
    _, grad, _, tg = ref(z[sane], ti[sane], tv[sane], 2.0)
    check_grad(dz[sane], grad, tg)
    p = torch.softmax(tv[0].double() / 2, 0)
    check_grad(dz[0], torch.zeros(vocab, device="cuda", dtype=torch.float64).scatter_add_(0, ti[0], -2 * p),
               torch.full((vocab,), 1e-5, device="cuda"))


def test_more_entries_than_outputs():
    """Every output named several times, in rows of every layout (a wave's, a workgroup's, slices)."""
    from lira_amd import distill_topk_loss_and_grad
    g = torch.Generator(device="cuda").manual_seed(8)
    for rows, vocab, top in ((5, 3, 60), (600, 2, 64), (7, 33, 500), (2, 20000, 700)):
        z = torch.randn(rows, vocab, generator=g, device="cuda")
        ti = torch.randint(0, min(vocab, 9), (rows, top), generator=g, device="cuda")
        tv = torch.randn(rows, top, generator=g, device="cuda")
        loss, grad, tl, tg = ref(z, ti, tv, 1.0)
        got, dz = distill_topk_loss_and_grad(z, ti, tv)
        # (an output named up to `top` times: that many additions more)
        check_loss(got, loss, tl + loss.abs() * top * 2.0 ** -24)
        check_grad(dz, grad, tg + top * 2.0 ** -24)


def test_teacher_lse():
    from lira_amd import distill_topk_loss, distill_topk_loss_and_grad
    g = torch.Generator(device="cuda").manual_seed(4)
    z, _, _, w = make(60, 900, 1)
    teacher = 2 * torch.randn(60, 900, generator=g, device="cuda")
    lse = torch.logsumexp(teacher.double() / 2, 1).float()
    tv, ti = torch.topk(teacher, 20, dim=1)
    loss, grad, tl, tg = ref(z, ti, tv, 2.0, lse)
    got, dz = distill_topk_loss_and_grad(z, ti, tv, 2.0, teacher_lse=lse)
    check_loss(got, loss, tl)
    check_grad(dz, grad, tg)
    z.requires_grad_(True)
    got = distill_topk_loss(z, ti, tv, 2.0, teacher_lse=lse, reduction="none")
    (dz,) = torch.autograd.grad(got, z, w)
    check_loss(got, loss, tl)
    check_grad(dz, grad * w.double()[:, None], tg * w.double().abs()[:, None] * 1.001)


def test_gradient_against_differences():
    """(f(z + h) - f(z - h)) / 2h: the third derivative of T^2 s logsumexp(z / T) is at most s / (10 T), so
    h = 1/16 leaves h^2 / 60 < 7e-5; a loss near 3 in fp32 is off by less than 2e-6, which gives 3e-5."""
    from lira_amd import distill_topk_loss, distill_topk_loss_and_grad
    z, ti, tv, _ = make(6, 33, 4, seed=9)
    z = z.clamp(-3, 3)
    h = 1 / 16
    _, dz = distill_topk_loss_and_grad(z, ti, tv)
    for v in range(33):
        e = torch.zeros_like(z)
        e[:, v] = h
        d = (distill_topk_loss(z + e, ti, tv, reduction="none") - distill_topk_loss(z - e, ti, tv, reduction="none")) / (2 * h)
        assert float((d - dz[:, v]).abs().max()) < 1e-4 + 5e-5


@pytest.mark.parametrize("dtype", list(DT))
def test_strides_shapes_and_in_place(dtype):
    from lira_amd import distill_topk_loss, distill_topk_loss_and_grad
    z, ti, tv, w = make(12, 501, 9, dtype)
    want, dwant = distill_topk_loss_and_grad(z, ti, tv, 2.0, row_weight=w)
    wide = torch.full((12, 517), 5.0, device="cuda", dtype=DT[dtype])
    wide[:, 7:508] = z
    loss, dz = distill_topk_loss_and_grad(wide[:, 7:508], ti, tv, 2.0, row_weight=w)
    assert torch.equal(loss, want) and torch.equal(dz, dwant)
    loss, dz = distill_topk_loss_and_grad(z.t().contiguous().t(), ti.t().contiguous().t(), tv.double().float(), 2.0, row_weight=w)
    assert torch.equal(loss, want) and torch.equal(dz, dwant)
    loss, dz = distill_topk_loss_and_grad(z.view(3, 4, 501), ti.view(3, 4, 9), tv.view(3, 4, 9), 2.0, row_weight=w.view(3, 4))
    assert torch.equal(loss.view(-1), want) and torch.equal(dz.view(12, 501), dwant)
    row = z[0].clone().requires_grad_(True)
    one = distill_topk_loss(row, ti[0], tv[0], 2.0, reduction="none")
    assert one.dim() == 0 and torch.equal(one.detach(), want[0])
    one.backward()
    # one row broadcast over several teachers: the gradients of its copies add up
    many = z[0].clone().requires_grad_(True)
    distill_topk_loss(many.expand(12, 501), ti, tv, 2.0, reduction="sum").backward()
    _, each = distill_topk_loss_and_grad(z[:1].expand(12, 501), ti, tv, 2.0)
    assert torch.allclose(many.grad.float(), each.float().sum(0), atol=12 * 2 * torch.finfo(DT[dtype]).eps, rtol=0)
    place = z.clone()
    loss, dz = distill_topk_loss_and_grad(place, ti, tv, 2.0, row_weight=w, grad_out=place)
    assert dz.data_ptr() == place.data_ptr() and torch.equal(loss, want) and torch.equal(place, dwant)


# (outputs of one vector or two more than a group's registers hold half of, in 16 bits and in 32)
@pytest.mark.parametrize("rows,vocab", [(3, 1), (3, 8), (3, 15), (5, 520), (5, 1032), (4100, 2056), (3, 4104), (200, 8200),
                                        (200, 16392), (195, 32776), (193, 65544), (5, 8200), (3, 16385), (7, 65544)])
@pytest.mark.parametrize("dtype", list(DT))
def test_rows_at_any_alignment(rows, vocab, dtype):
    from lira_amd import distill_topk_loss, distill_topk_loss_and_grad
    z, ti, tv, w = make(rows, vocab, min(vocab, 7), dtype, seed=vocab)
    ti[:, 0] = 0
    ti[1:, -1] = vocab - 1
    loss, grad, tl, tg = ref(z, ti, tv, 2.0)
    for off, goff in ((1, 1), (3, 3), (7, 0), (0, 5)):
        zs = torch.cat([z.new_zeros(off), z.flatten()])[off:].view(rows, vocab)
        room = torch.full((goff + rows * vocab + 9,), 77.0, device="cuda", dtype=DT[dtype])
        got, dz = distill_topk_loss_and_grad(zs, ti, tv, 2.0, row_weight=w, grad_out=room[goff:goff + rows * vocab].view(rows, vocab))
        check_loss(got, loss, tl)
        check_grad(dz, grad * w.double()[:, None], tg * w.double().abs()[:, None] * 1.001)
        assert bool((room[:goff] == 77).all()) and bool((room[goff + rows * vocab:] == 77).all())
    zs.requires_grad_(True)
    got = distill_topk_loss(zs, ti, tv, 2.0, reduction="none")
    check_loss(got, loss, tl)
    (dz,) = torch.autograd.grad(got, zs, w)
    check_grad(dz, grad * w.double()[:, None], tg * w.double().abs()[:, None] * 1.001)


@pytest.mark.parametrize("rows,vocab", [(2, 131072), (300, 4000), (4096, 64)])
def test_repeats_bit_for_bit_on_streams_and_in_graphs(rows, vocab):
    from lira_amd import distill_topk_loss_and_grad
    sets = [make(rows, vocab, 16, "bf16", seed=i, masked=True) for i in range(3)]
    want = [distill_topk_loss_and_grad(z, ti, tv, 2.0, row_weight=w) for z, ti, tv, w in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [distill_topk_loss_and_grad(z, ti, tv, 2.0, row_weight=w, stream=side) for z, ti, tv, w in sets]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    now = [x.clone() for x in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dz = distill_topk_loss_and_grad(*now[:3], 2.0, row_weight=now[3])
    for i in (1, 2, 0, 1):
        for a, b in zip(now, sets[i]):
            a.copy_(b)
        graph.replay()
        again = distill_topk_loss_and_grad(*sets[i][:3], 2.0, row_weight=sets[i][3])
        torch.cuda.synchronize()
        assert torch.equal(loss, want[i][0]) and torch.equal(dz, want[i][1]) and torch.equal(again[1], dz)


def test_more_than_2_31_elements():
    from lira_amd import distill_topk_loss_and_grad
    rows, vocab = (1 << 31) // 65536 + 9, 65536
    z, ti, tv, _ = make(4, vocab, 12, "bf16")
    big = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    big[-4:] = z
    bi = torch.full((rows, 12), -1, device="cuda")
    bi[-4:] = ti
    bt = torch.zeros(rows, 12, device="cuda")
    bt[-4:] = tv
    loss, dz = distill_topk_loss_and_grad(big, bi, bt)
    a, b = distill_topk_loss_and_grad(z, ti, tv)
    assert not loss[:-4].any() and not dz[:-4].any()
    assert torch.equal(loss[-4:], a) and torch.equal(dz[-4:], b)


def test_refusals():
    from lira_amd import LiraError, distill_topk_loss, distill_topk_loss_and_grad
    z, ti, tv, w = make(4, 50, 6)
    for args, kw, text in (((z.double(), ti, tv), {}, "float32"), ((z, ti.short(), tv), {}, "int32"), ((z, ti, tv.double()), {}, "float32"),
                           ((z, ti[:3], tv), {}, "leading"), ((z, ti[:, :5], tv), {}, "same"), ((z, ti[:, :0], tv[:, :0]), {}, "at least one"),
                           ((z, ti.cpu(), tv), {}, "cuda"), ((z[:, :0], ti, tv), {}, "output"), ((z, ti, tv, 0.0), {}, "temperature"),
                           ((z, ti, tv, -1.0), {}, "temperature"), ((z, ti, tv), {"teacher_lse": w[:3]}, "teacher_lse")):
        for f in (distill_topk_loss, distill_topk_loss_and_grad):
            with pytest.raises(ValueError, match=text):
                f(*args, **kw)
    for kw in ({"row_weight": w[:3]}, {"grad_out": z[:3]}, {"grad_out": z.half()}, {"grad_out": z.t()}):
        with pytest.raises(ValueError, match=next(iter(kw))):
            distill_topk_loss_and_grad(z, ti, tv, **kw)
    with pytest.raises(LiraError, match="top must be at most 1024"):
        distill_topk_loss_and_grad(torch.zeros(1, 2000, device="cuda"), torch.zeros(1, 1025, dtype=torch.int64, device="cuda"),
                                   torch.zeros(1, 1025, device="cuda"))
