"""Calls that write a tensor through its address tell autograd so: a graph
that saved the tensor refuses its backward pass, as after torch's own
in-place operations, instead of giving the gradient at other values."""
import pytest

pytestmark = pytest.mark.gpu


def rows(torch, N=4, V=500, K=3):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(N, V, generator=g, device="cuda")
    ids = torch.randint(0, V, (N, K), generator=g, device="cuda", dtype=torch.int32)
    t = torch.randn(N, K, generator=g, device="cuda")
    return x, ids, t


def writers(torch, pz, x, ids, t):
    """(what is called, what it writes) of each call."""
    N, V = x.shape
    loss, stats = torch.empty(N, device="cuda"), torch.empty(N, 4, device="cuda")
    grad, out = torch.empty_like(x), torch.empty_like(x)
    n = torch.empty(N, dtype=torch.int32, device="cuda")
    q, wq = (torch.zeros(r, 512, dtype=torch.int8, device="cuda")[:, :V] for r in (N, 7))
    s, ws, logits = torch.ones(N, device="cuda"), torch.ones(7, device="cuda"), torch.empty(N, 7, device="cuda")
    pz.distill_forward(x, ids, t, loss, stats)
    return {
        "process apart": (lambda: pz.process_logits(x, out, n_allowed=n), (out, n)),
        "process in place": (lambda: pz.process_logits(x), (x,)),
        "forward": (lambda: pz.distill_forward(x, ids, t, loss, stats), (loss, stats)),
        "forward alone": (lambda: pz.distill_forward(x, ids, t, loss), (loss,)),
        "backward": (lambda: pz.distill_backward(x, ids, t, stats, grad), (grad,)),
        "both": (lambda: pz.distill_loss_grad(x, ids, t, loss, grad), (loss, grad)),
        "quantize": (lambda: pz.quantize_rows_i8(x, q, s), (q, s)),
        "product": (lambda: pz.matmul_i8(q, s, wq, ws, logits), (logits,)),
        "head": (lambda: pz.lm_head_i8(x, wq, ws, logits, q, s), (logits, q, s)),
    }


def test_what_is_written_counts_as_changed(cuda, pz):
    torch = cuda
    x, ids, t = rows(torch)
    calls = writers(torch, pz, x, ids, t)
    watched = {id(v): v for _, outs in calls.values() for v in outs}
    watched.update((id(v), v) for v in (x, ids, t))
    for name, (call, outs) in calls.items():
        before = {k: v._version for k, v in watched.items()}
        call()
        for k, v in watched.items():
            assert (v._version > before[k]) == any(v is o for o in outs), name


@pytest.mark.parametrize("how", ["process", "both", "backward"])
def test_a_backward_pass_over_changed_logits_is_refused(cuda, pz, how):
    """distill_loss saves its logits; each call writes over them before the
    backward pass.  Through a view too: it shares its base's version."""
    torch = cuda
    for view in (False, True):
        x, ids, t = rows(torch)
        leaf = x.clone().requires_grad_(True)
        logits = leaf * 1
        loss = pz.distill_loss(logits, ids, t)
        at = logits.detach()[:, :] if view else logits.detach()
        one, stats = torch.empty(4, device="cuda"), torch.empty(4, 4, device="cuda")
        if how == "process":
            pz.process_logits(at, cfg=None, mask=torch.zeros(4, 16, dtype=torch.int32, device="cuda"))
        elif how == "both":
            pz.distill_loss_grad(at, ids, t, one, at)
        else:
            pz.distill_forward(at, ids, t, one, stats)
            pz.distill_backward(at, ids, t, stats, at)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.sum().backward()


def test_unchanged_logits_and_inference_tensors_pass(cuda, pz):
    torch = cuda
    x, ids, t = rows(torch)
    leaf = x.clone().requires_grad_(True)
    loss = pz.distill_loss(leaf, ids, t)
    pz.process_logits(leaf.detach(), torch.empty_like(x))  # reads them only
    loss.sum().backward()
    want, grad = torch.empty(4, device="cuda"), torch.empty_like(x)
    pz.distill_loss_grad(x, ids, t, want, grad)
    assert torch.equal(loss.detach(), want) and torch.allclose(leaf.grad, grad, rtol=1e-5, atol=1e-9)
    with torch.inference_mode():  # such tensors have no version
        y = x.clone()
        pz.process_logits(y)
        for name, (call, _) in writers(torch, pz, y, ids, t).items():
            call()
    assert torch.isfinite(want).all()
