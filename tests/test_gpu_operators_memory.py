"""GPU: what the 4-bit and distillation operators read and write, as other parts of a program see it: copies of
packed rows, outputs that autograd has saved, shared memory, streams, modules' state."""
import copy
import io
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def saved(t):
    f = io.BytesIO()
    torch.save(t, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t)), saved])
def test_copies_outlive_their_original(how):
    from lira_amd import IndexMX4, mx4_linear, mx4_matmul, mx4_quantize
    x, q = torch.randn(70, 300, generator=gen(1), device="cuda"), torch.randn(20, 300, generator=gen(2), device="cuda")
    t = mx4_quantize(x)
    want = [t.dequantize(), mx4_linear(q, t), mx4_matmul(mx4_quantize(q), t), t[5:9].dequantize()]
    c, part = how(t), how(t[5:9])
    t.codes.zero_()  # (what the original's memory may hold once it is gone)
    t.scales.zero_()
    del t
    got = [c.dequantize(), mx4_linear(q, c), mx4_matmul(mx4_quantize(q), c), part.dequantize()]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    idx = IndexMX4(300)
    idx.add(x)
    D, I = idx.search(q, 5)
    other = how(idx)
    idx._packed().codes.zero_()
    idx._packed().scales.zero_()
    D2, I2 = other.search(q, 5)
    assert torch.equal(D, D2) and torch.equal(I, I2)


def student(rows=6, vocab=50, top=4, seed=3):
    g = gen(seed)
    y = torch.randn(rows, vocab, generator=g, device="cuda", requires_grad=True)
    tv, ti = torch.topk(torch.randn(rows, vocab, generator=g, device="cuda"), top, dim=1)
    return y, ti, tv


@pytest.mark.parametrize("f", [torch.tanh, torch.sigmoid, torch.exp])
@pytest.mark.parametrize("detached", [False, True])
def test_gradient_over_saved_logits_is_seen_by_autograd(f, detached):
    """The logits are what f saved for its backward pass: once they are overwritten that pass must not run on them."""
    from lira_amd import distill_topk_loss_and_grad
    y, ti, tv = student()
    z = f(y)
    was = z._version
    _, dz = distill_topk_loss_and_grad(z, ti, tv, grad_out=z.detach() if detached else z)
    assert z._version > was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward(dz.detach().clone())


def test_gradient_over_logits_that_nobody_saved():
    """A layer saves its inputs, not its outputs: its backward pass runs on the gradient in the logits' place."""
    from lira_amd import distill_topk_loss_and_grad
    y, ti, tv = student()
    w = torch.randn(50, 50, generator=gen(9), device="cuda")
    z = y @ w
    _, dz = distill_topk_loss_and_grad(z.detach().clone(), ti, tv)
    want = torch.autograd.grad(z, y, dz)[0]
    z = y @ w
    _, dz = distill_topk_loss_and_grad(z, ti, tv, grad_out=z)
    assert dz is z
    assert torch.equal(torch.autograd.grad(z, y, dz.detach())[0], want)


def test_outputs_of_products_are_seen_by_autograd():
    from lira_amd import mx4_linear, mx4_matmul, mx4_quantize
    x = torch.randn(6, 64, generator=gen(4), device="cuda")
    w = mx4_quantize(torch.randn(50, 64, generator=gen(5), device="cuda"))
    calls = [lambda out: mx4_linear(x, w, out=out), lambda out: mx4_matmul(mx4_quantize(x), w, out=out),
             lambda out: w[:6].dequantize(out=out)]
    for call, cols in zip(calls, (50, 50, 64)):
        y = torch.randn(6, cols, generator=gen(6), device="cuda", requires_grad=True)
        z = torch.tanh(y)
        call(z.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        out = torch.zeros(8, cols, device="cuda")
        was = out._version
        call(out[1:7])  # (a view's base too)
        assert out._version > was
        with torch.inference_mode():
            inside = torch.zeros(6, cols, device="cuda")
            call(inside)
        again = inside.clone()
        call(inside)
        assert torch.equal(inside, again)


def test_gradient_may_share_memory_with_the_logits_alone():
    """Workgroups still read what lies elsewhere: only the logits' own places are each read before they are written."""
    from lira_amd import distill_topk_loss_and_grad
    rows, vocab, top = 6, 64, 8
    g = gen(8)
    buf = torch.randn(rows + 1, vocab, generator=g, device="cuda")
    tv, ti = torch.topk(torch.randn(rows, vocab, generator=g, device="cuda"), top, dim=1)
    ti = ti.int()
    w, lse = torch.rand(rows, generator=g, device="cuda"), torch.logsumexp(tv, 1)
    z = buf[:-1]
    keep = buf.clone()
    flat = torch.zeros(4 * rows * vocab, device="cuda")
    cases = [
        (z, ti, tv, {"grad_out": buf[1:]}),
        (buf[1:], ti, tv, {"grad_out": buf[:-1]}),
        (z.flatten()[8:], ti.flatten()[:4], tv.flatten()[:4], {"grad_out": z.flatten()[:-8]}),
        (buf.as_strided((3, vocab), (2 * vocab, 1)), ti[:3], tv[:3], {"grad_out": buf[:3]}),  # (rows further apart)
        (z, flat[:rows * top].view(torch.int32).view(rows, top), tv, {"grad_out": flat[:rows * vocab].view(rows, vocab)}),
        (z, ti, flat[rows * vocab - 1:rows * vocab - 1 + rows * top].view(rows, top), {"grad_out": flat[:rows * vocab].view(rows, vocab)}),
        (z, ti, tv, {"row_weight": flat[5:5 + rows], "grad_out": flat[:rows * vocab].view(rows, vocab)}),
        (z, ti, tv, {"teacher_lse": flat[5:5 + rows], "grad_out": flat[:rows * vocab].view(rows, vocab)}),
    ]
    for zz, ii, tt, kw in cases:
        with pytest.raises(ValueError, match="share memory"):
            distill_topk_loss_and_grad(zz, ii, tt, **kw)
    assert torch.equal(buf, keep) and not flat.any()
    # what only looks alike: the logits themselves, the memory behind an input's end, inputs that are copied on the way
    want, dwant = distill_topk_loss_and_grad(z, ti, tv, teacher_lse=lse, row_weight=w)
    at = flat[rows * vocab:2 * rows * vocab].view(rows, vocab)
    flat[:rows * vocab].view(rows, vocab).copy_(z)
    loss, dz = distill_topk_loss_and_grad(flat[:rows * vocab].view(rows, vocab), ti, tv, teacher_lse=lse, row_weight=w, grad_out=at)
    assert torch.equal(loss, want) and torch.equal(dz, dwant)
    t = z.t().contiguous()
    loss, dz = distill_topk_loss_and_grad(t.t(), ti, tv, teacher_lse=lse, row_weight=w, grad_out=t.view(rows, vocab))
    assert torch.equal(loss, want) and torch.equal(dz, dwant)
    own = z.clone()
    for view in (own, own.view(2, 3, vocab)):
        own.copy_(z)
        lead = view.shape[:-1]
        loss, dz = distill_topk_loss_and_grad(view, ti.view(*lead, top), tv.view(*lead, top), teacher_lse=lse.view(lead),
                                              row_weight=w.view(lead), grad_out=view)
        assert torch.equal(loss.flatten(), want) and torch.equal(own, dwant)


def prober(seed=0, nb=16, d=32):
    from lira_amd.probing import MLP_2_Input
    torch.manual_seed(seed)
    return MLP_2_Input(nb, d, nb).cuda()


def test_packed_prober_refuses_a_model_with_more_layers():
    """Layers that it would leave out: the scores would be another model's."""
    from lira_amd.probing import MX4Probe
    deeper = prober()
    deeper.fc = torch.nn.Sequential(*list(deeper.fc)[:2], torch.nn.Linear(deeper.fc[2].in_features, 16), torch.nn.ReLU(),
                                    torch.nn.Linear(16, 16), torch.nn.Sigmoid()).cuda()
    with pytest.raises(ValueError, match="MLP_2_Input"):
        MX4Probe(deeper)
    normed = prober()
    normed.vector_net.add_module("4", torch.nn.BatchNorm1d(normed.vector_net[2].out_features).cuda())
    with pytest.raises(ValueError, match="MLP_2_Input"):
        MX4Probe(normed)


def test_packed_prober_has_its_weights_in_its_state():
    from lira_amd.probing import MX4Probe
    xd, q = torch.randn(50, 16, generator=gen(1), device="cuda"), torch.randn(50, 32, generator=gen(2), device="cuda")
    probe, other = MX4Probe(prober(0)), MX4Probe(prober(1))
    want = probe(xd, q)
    assert not torch.equal(other(xd, q), want)
    state = probe.state_dict()
    assert len(state) == 18 and {v.dtype for v in state.values()} == {torch.uint8, torch.float32}
    other.load_state_dict(state)
    assert torch.equal(other(xd, q), want)
    other.load_state_dict({k: v.clone() for k, v in state.items()}, assign=True)
    assert torch.equal(other(xd, q), want)
    for again in (copy.deepcopy(probe), pickle.loads(pickle.dumps(probe)), saved(probe)):
        for v in other.state_dict().values():
            v.zero_()
        assert torch.equal(again(xd, q), want)
    away = copy.deepcopy(probe).cpu()
    assert all(v.device.type == "cpu" for v in away.state_dict().values())
    with pytest.raises(ValueError, match="GPU|cpu"):
        away(xd, q)
    with pytest.raises(ValueError, match="GPU|cpu"):
        away(xd.cpu(), q.cpu())
    assert torch.equal(away.to("cuda")(xd, q), want)
    assert torch.equal(probe(xd, q), want)


def stream_calls():
    """name -> (inputs of the current stream, the call that reads them on another one)"""
    from lira_amd import distill_topk_loss_and_grad, mx4_dequantize, mx4_linear, mx4_matmul, mx4_quantize
    g = gen(12)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    rows = 3000  # (of a size that the allocator gives to nothing else here)
    ids = torch.randint(0, 500, (rows, 70), generator=g, device="cuda")
    w = mx4_quantize(normal(700, 500))
    return {
        "quantize": ([normal(rows, 500)], lambda s, x: mx4_quantize(x, stream=s)),
        "quantize columns": ([normal(500, rows)], lambda s, x: mx4_quantize(x.t(), stream=s)),
        "dequantize": ([mx4_quantize(normal(rows, 500))], lambda s, t: mx4_dequantize(t, stream=s)),
        "dequantize out": ([normal(700, 500)], lambda s, out: w.dequantize(out=out, stream=s)),
        "linear": ([normal(rows, 500), mx4_quantize(normal(700, 500)), normal(700).half()],
                   lambda s, x, w, b: mx4_linear(x, w, b, stream=s)),
        "matmul": ([mx4_quantize(normal(rows, 500)), mx4_quantize(normal(700, 500)), normal(700)],
                   lambda s, a, b, c: mx4_matmul(a, b, c, stream=s)),
        "linear out": ([normal(rows, 700)], lambda s, out, x=normal(rows, 500): mx4_linear(x, w, out=out, stream=s)),
        "distill": ([normal(rows, 500), ids, normal(rows, 70), normal(rows), normal(rows)],
                    lambda s, z, i, t, lse, wt: distill_topk_loss_and_grad(z, i, t, 1.0, lse, wt, stream=s)),
        "distill out": ([normal(rows, 500)], lambda s, dz, z=normal(rows, 500), t=normal(rows, 70):
                        distill_topk_loss_and_grad(z, ids, t, grad_out=dz, stream=s)),
    }


@pytest.mark.parametrize("name", ["quantize", "quantize columns", "dequantize", "dequantize out", "linear", "matmul", "linear out",
                                  "distill", "distill out"])
def test_memory_read_on_another_stream_is_not_given_out_again(name):
    """An input that is dropped right after the call: its stream's allocator must not hand its memory out while the
    other stream has work that reads it (looked at by address: nothing writes there)."""
    from lira_amd import MX4Tensor
    side = torch.cuda.Stream()
    inputs, call = stream_calls()[name]
    call(side, *inputs)  # (its kernels are loaded)
    torch.cuda.synchronize()
    inputs, call = stream_calls()[name]
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(500_000_000)  # (0.2 s; the call waits behind it)
    kept = []
    result = call(side, *inputs)
    held = [b for t in inputs for b in ((t._buf,) if isinstance(t, MX4Tensor) and t._buf is not None else
                                        (t.codes, t.scales) if isinstance(t, MX4Tensor) else (t,))]
    spans = [(b.untyped_storage().data_ptr(), b.untyped_storage().nbytes()) for b in held]
    del inputs, call, held
    for at, size in spans:
        kept += [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
    pending = not side.query()
    for new in kept:
        for at, size in spans:
            assert new.data_ptr() + new.numel() <= at or at + size <= new.data_ptr()
    assert pending  # (else the test has looked too late)
    torch.cuda.synchronize()
    del result
