"""GPU: distillation's teacher entries where they can go wrong: rows masked whole, entries that stand for nothing,
many entries of one output, tensors that saved-tensor hooks bring back in another layout."""
import pytest
import torch

from test_gpu_distill import INF, check_grad, check_loss, make, ref

pytestmark = pytest.mark.gpu


def both(z, ti, tv, t, lse=None):
    """Losses and gradients by every path: in one call, and the backward pass of its own."""
    from lira_amd import distill_topk_loss, distill_topk_loss_and_grad
    out = [distill_topk_loss_and_grad(z, ti, tv, t, teacher_lse=lse)]
    zg = z.clone().requires_grad_(True)
    loss = distill_topk_loss(zg, ti, tv, t, teacher_lse=lse, reduction="none")
    (dz,) = torch.autograd.grad(loss, zg, torch.ones_like(loss))
    return out + [(loss.detach(), dz)]


# (a wave's rows, a workgroup's, slices; lists of up to 64 entries and longer ones)
@pytest.mark.parametrize("rows,vocab,top", [(20, 40, 5), (30, 9000, 20), (6, 100000, 30), (20, 400, 90), (700, 300, 8)])
def test_rows_of_a_masked_teacher_with_its_own_lse(rows, vocab, top):
    """logsumexp of a row that is masked whole is -inf: no entry counts, so loss and gradient are 0."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    z = 2 * torch.randn(rows, vocab, generator=g, device="cuda")
    teacher = 2 * torch.randn(rows, vocab, generator=g, device="cuda")
    teacher[1::3] = -INF
    teacher[2, 1:] = -INF
    lse = torch.logsumexp(teacher / 2, 1)
    tv, ti = torch.topk(teacher, top, dim=1)
    assert float(lse[1]) == -INF
    some = torch.ones(rows, dtype=torch.bool, device="cuda")
    some[1::3] = False
    want, grad, tl, tg = ref(z[some], ti[some], tv[some], 2.0, lse[some])
    z[4] = float("nan")  # (of no consequence: no entry counts)
    for loss, dz in both(z, ti, tv, 2.0, lse):
        assert not loss[~some].any() and not dz[~some].any()
        check_loss(loss[some], want, tl)
        check_grad(dz[some], grad, tg)


@pytest.mark.parametrize("rows,vocab,top", [(50, 40, 64), (50, 5000, 64), (4, 60000, 200), (30, 700, 1024)])
def test_entries_padded_with_a_logit_of_minus_infinity(rows, vocab, top):
    """Short lists filled up with id 0 and a logit of -inf: as if the rest were unused."""
    z, ti, tv, _ = make(rows, vocab, min(top, vocab // 2), seed=top)
    n = torch.randint(0, min(top, vocab // 2, 9), (rows, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    pad = top - ti.shape[1]
    ti = torch.nn.functional.pad(ti, (0, pad))
    tv = torch.nn.functional.pad(tv, (0, pad))
    gone = torch.arange(top, device="cuda") >= n
    padded = both(z, ti.masked_fill(gone, 0), tv.masked_fill(gone, -INF), 2.0)
    unused = both(z, ti.masked_fill(gone, -1), tv, 2.0)
    for a, b in zip(padded, unused):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("rows,vocab,top,ids", [(3, 2000, 1024, 1), (3, 100000, 1024, 1), (5, 4000, 64, 1), (9, 4000, 700, 3),
                                                (4, 70000, 1024, 8), (600, 1000, 64, 2), (4, 300000, 1024, 1000)])
def test_many_entries_of_one_output(rows, vocab, top, ids):
    """All entries name the same few outputs, next to each other: one thread stores them all."""
    g = torch.Generator(device="cuda").manual_seed(top + ids)
    z = torch.randn(rows, vocab, generator=g, device="cuda")
    ti = vocab // 3 + torch.randint(0, ids, (rows, top), generator=g, device="cuda")
    tv = torch.randn(rows, top, generator=g, device="cuda")
    loss, grad, tl, tg = ref(z, ti, tv, 1.0)
    # (an output named up to `top` times: that many additions more, of at most 1 in all)
    for got, dz in both(z, ti, tv, 1.0):
        check_loss(got, loss, tl + loss.abs() * top * 2.0 ** -24)
        check_grad(dz, grad, tg + top * 2.0 ** -24)


def test_what_hooks_bring_back_in_another_layout():
    """Saved-tensor hooks may return the same values in tensors that are laid out otherwise."""
    from lira_amd import distill_topk_loss
    z, ti, tv, w = make(30, 800, 9, "fp32")
    lse = torch.logsumexp(z, 1)
    z.requires_grad_(True)

    def step():
        (g,) = torch.autograd.grad(distill_topk_loss(z, ti, tv, 2.0, teacher_lse=lse, reduction="none"), z, w)
        return g

    def spread(t):
        return torch.stack((t, t), -1)[..., 0]  # (every second element of twice the memory)

    want = step()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        got = step()
    assert torch.equal(got, want)


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("change", [lambda t: t.half(), lambda t: t[:-1], lambda t: t.cpu(), lambda t: t.flatten()])
def test_what_hooks_bring_back_as_another_tensor(which, change):
    """Another type, size or device than was saved: refused, not read as if it were the same."""
    from lira_amd import distill_topk_loss
    z, ti, tv, _ = make(30, 800, 9, "fp32")
    lse = torch.logsumexp(z, 1)
    if which == 3 and change(lse).shape == lse.shape and change(lse).dtype == lse.dtype and change(lse).is_cuda:
        pytest.skip("this change leaves a vector as it is")
    z.requires_grad_(True)
    count = iter(range(5))  # (saved in the order logits, ids, teacher, its logsumexp, statistics)

    def unpack(t):
        return change(t) if next(count) == which else t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        loss = distill_topk_loss(z, ti, tv, 2.0, teacher_lse=lse)
    with pytest.raises(RuntimeError, match="came back"):
        loss.backward()
