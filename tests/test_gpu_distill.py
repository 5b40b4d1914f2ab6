"""pz_distill_* against numpy in fp64, within bounds derived from the kernels'
fp32 steps (rows_ref.distill_row)."""
import numpy as np
import pytest

from rows_ref import bf16_round, close, distill_row

pytestmark = pytest.mark.gpu

LOWEST = -np.finfo(np.float32).max


def make(seed, N, V, K, rest, *, odd=True):
    """Student rows, lists, weights; with `odd`, ignored and repeated ids,
    lists that end early, rows without a weight or a list."""
    r = np.random.default_rng(seed)
    x = (r.standard_normal((N, V)) * 3).astype(np.float32)
    ids = np.stack([r.permutation(V)[:K] if V < 200000 else r.choice(V, K, replace=False) for _ in range(N)]).astype(np.int32)
    np.put_along_axis(x, ids, np.take_along_axis(x, ids, 1) + (r.random((N, K)) * 6).astype(np.float32), 1)
    t = (r.standard_normal((N, K)) * 2).astype(np.float32)
    if rest:
        t = (t - np.log(np.exp(t.astype(np.float64)).sum(1, keepdims=True)) + np.log(
            1 - 0.4 * r.random((N, 1)))).astype(np.float32)
    n = np.full(N, K, dtype=np.int32)
    w = (0.5 + r.random(N)).astype(np.float32)
    if odd and N >= 6:
        n[1], n[2] = max(1, K // 2), 0
        w[3] = 0.0
        if K > 2:
            ids[4, 1] = -1
            ids[4, 2] = V
            ids[5, K - 1] = ids[5, 0]  # an id listed twice, its probabilities add
            t[5, K - 1] -= 1.0
            t[5, 1] = -np.inf
    return x, ids, t, n, w


def run(torch, pz, x, ids, t, n, w, T, rest, dtype, up=None, how="both", gap=0, lead=0, inplace=False):
    """Losses and gradients of the calls, as numpy."""
    N, V = x.shape
    buf = torch.full((lead + (N + 1) * (V + gap),), 7.0, dtype=dtype, device="cuda")
    xs = buf[lead:lead + N * (V + gap)].view(N, V + gap)[:, :V]
    xs.copy_(torch.from_numpy(x).cuda().to(dtype))
    gbuf = buf if inplace else torch.full((lead + 1 + (N + 1) * (V + gap),), 7.0, dtype=dtype, device="cuda")
    first = lead if inplace else lead + (1 if gap else 0)
    g = gbuf[first:first + N * (V + gap)].view(N, V + gap)[:, :V]
    dev = [torch.from_numpy(a).cuda() for a in (ids, t, n, w)]
    kw = dict(weight=dev[3], temperature=T, mode=pz.DISTILL_REST if rest else pz.DISTILL_LIST, n_list=dev[2])
    loss = torch.full((N + 1,), -9.0, device="cuda")
    if how == "one":
        pz.distill_loss_grad(xs, dev[0], dev[1], loss, g, **kw)
    else:
        stats = torch.empty(N, 4, device="cuda")
        pz.distill_forward(xs, dev[0], dev[1], loss, stats, **kw)
        pz.distill_backward(xs, dev[0], dev[1], stats, g, None if up is None else torch.from_numpy(up).cuda(), **kw)
    torch.cuda.synchronize()
    assert float(loss[N]) == -9.0
    rest_of = torch.ones(gbuf.numel(), dtype=torch.bool, device="cuda")
    rest_of[first:first + N * (V + gap)].view(N, V + gap)[:, :V] = False
    assert bool((gbuf[rest_of] == 7).all())
    return loss[:N].cpu().numpy(), g.float().cpu().numpy()


def check(x, ids, t, n, w, T, rest, loss, grad, half, up=None):
    for i in range(x.shape[0]):
        l, g, dl, dg = distill_row(x[i], ids[i, :n[i]], t[i, :n[i]], T, rest, float(w[i]))
        u = 1.0 if up is None else float(up[i])
        assert close(loss[i], l, dl), (i, loss[i], l, dl)
        assert close(grad[i], g * u, dg * abs(u), half + 2.0 ** -23), (
            i, np.nanmax(np.abs(grad[i] - g * u)), np.nanmax(dg))


SHAPES = [
    # N, V, K, extra elements between rows, in front
    (6, 1, 1, 0, 0), (6, 7, 3, 1, 1), (6, 33, 33, 0, 0), (7, 1000, 20, 0, 0), (6, 4099, 64, 5, 3),
    (6, 32000, 1024, 0, 0), (6, 70001, 50, 0, 1), (8, 128256, 20, 0, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rest", [False, True], ids=["list", "rest"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("T", [1.0, 2.5, 0.5])
def test_loss_and_gradient(cuda, pz, shape, rest, dtype, T):
    torch = cuda
    N, V, K, gap, lead = shape
    x, ids, t, n, w = make(V + K, N, V, K, rest)
    td, half = (torch.float32, 2.0 ** -24) if dtype == "f32" else (torch.bfloat16, 2.0 ** -8)
    if dtype == "bf16":
        x = bf16_round(x)
    up = (np.random.default_rng(1).random(N) * 2 - 0.5).astype(np.float32)
    a = run(torch, pz, x, ids, t, n, w, T, rest, td, up, gap=gap, lead=lead)
    check(x, ids, t, n, w, T, rest, *a, half, up)
    b = run(torch, pz, x, ids, t, n, w, T, rest, td, how="one", gap=gap, lead=lead)
    check(x, ids, t, n, w, T, rest, *b, half)
    assert np.array_equal(a[0], b[0], equal_nan=True)
    for how in ("both", "one"):  # the gradient over the logits themselves
        c = run(torch, pz, x, ids, t, n, w, T, rest, td, how=how, gap=gap, lead=lead, inplace=True)
        check(x, ids, t, n, w, T, rest, *c, half)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_longer_than_the_registers_hold(cuda, pz, dtype):
    """Rows beyond 8 CTAs x 64 KB are read twice."""
    torch = cuda
    N, V = 2, 600001
    x, ids, t, n, w = make(3, N, V, 30, True, odd=False)
    td, half = (torch.float32, 2.0 ** -24) if dtype == "f32" else (torch.bfloat16, 2.0 ** -8)
    if dtype == "bf16":
        x = bf16_round(x)
    for how, inplace in (("one", False), ("one", True), ("both", False)):
        got = run(torch, pz, x, ids, t, n, w, 1.0, True, td, how=how, inplace=inplace)
        check(x, ids, t, n, w, 1.0, True, *got, half)


@pytest.mark.parametrize("rest", [False, True], ids=["list", "rest"])
def test_the_longest_rows_and_lists(cuda, pz, rest):
    torch = cuda
    N, V, K = 2, 1 << 20, 1024
    x, ids, t, n, w = make(31, N, V, K, rest, odd=False)
    for how, inplace in (("one", True), ("both", False)):
        got = run(torch, pz, x, ids, t, n, w, 1.0, rest, torch.float32, how=how, inplace=inplace)
        check(x, ids, t, n, w, 1.0, rest, *got, 2.0 ** -24)


@pytest.mark.parametrize("rest", [False, True], ids=["list", "rest"])
@pytest.mark.parametrize("shape", [(9, 5, 12), (6, 40, 300), (4, 3000, 1024)], ids=str)
def test_ids_listed_many_times(cuda, pz, shape, rest):
    """Lists longer than the vocabulary, ids that repeat and leave it; the
    last row lists one id only."""
    torch = cuda
    N, V, K = shape
    r = np.random.default_rng(K)
    x = (r.standard_normal((N, V)) * 3).astype(np.float32)
    ids = r.integers(-2, V + 2, (N, K)).astype(np.int32)
    ids[N - 1] = 1
    t = r.standard_normal((N, K)).astype(np.float32)
    if rest:  # the mass of the ids that count stays below one
        t = (t - np.log(np.exp(t.astype(np.float64)).sum(1, keepdims=True)) - 0.2).astype(np.float32)
    n, w = np.full(N, K, np.int32), np.ones(N, np.float32)
    for how in ("one", "both"):
        got = run(torch, pz, x, ids, t, n, w, 1.0, rest, torch.float32, how=how)
        check(x, ids, t, n, w, 1.0, rest, *got, 2.0 ** -24)


@pytest.mark.parametrize("rest", [False, True], ids=["list", "rest"])
def test_values_at_the_edges(cuda, pz, rest):
    torch = cuda
    N, V, K = 14, 5000, 8
    x, ids, t, n, w = make(17, N, V, K, rest, odd=False)
    x[0] = -np.inf                          # no distribution
    x[1] = LOWEST                           # flat, at the type's lowest value
    x[2, :4000] = -np.inf                   # masked places
    x[2, ids[2]] = 1.0
    x[3, ids[3, 0]] = -np.inf               # a listed id the student excludes
    x[4, 17] = np.nan
    x[5, 17] = np.inf
    t[6] = -np.inf                          # the teacher gives the list nothing
    t[7, 2] = np.nan
    x[8] = LOWEST
    x[8, ids[8, 1]] = 3.0                   # masked by the lowest value but for one id
    x[9] -= 400.0                           # off the list next to nothing
    x[9, ids[9]] = 10.0
    w[10] = 0.0
    x[10] = np.nan                          # padding may hold anything
    n[11] = 0
    x[11] = np.nan
    x[12, ids[12]] = -300.0                 # on the list next to nothing
    w[13] = -1.0
    for how in ("both", "one"):
        loss, grad = run(torch, pz, x, ids, t, n, w, 1.0, rest, torch.float32, how=how)
        check(x, ids, t, n, w, 1.0, rest, loss, grad, 2.0 ** -24)
    assert loss[0] == np.inf and not grad[0].any()
    assert np.isfinite(loss[9]) and loss[10] == 0 and not grad[10].any() and loss[11] == 0


def test_a_list_of_the_whole_vocabulary(cuda, pz):
    torch = cuda
    N, V = 6, 40
    x, ids, t, n, w = make(8, N, V, V, True, odd=False)
    for i in range(N):  # log-probabilities that sum to 1 but for rounding
        t[i] = (t[i] - np.log(np.exp(t[i].astype(np.float64)).sum())).astype(np.float32)
    loss, grad = run(torch, pz, x, ids, t, n, w, 1.0, True, torch.float32)
    assert np.isfinite(loss).all()
    check(x, ids, t, n, w, 1.0, True, loss, grad, 2.0 ** -24)


@pytest.mark.parametrize("rest", [False, True], ids=["list", "rest"])
def test_gradient_against_differences(cuda, pz, rest):
    """Central differences of the loss in single logits.  With steps of
    h = 2^-5 and third derivatives of a log-softmax below 1 the difference is
    off by h^2 / 6 < 1.7e-4, and the two losses' bounds by (d1 + d2) / 2h."""
    torch = cuda
    V, K, h, T = 300, 10, 2.0 ** -5, 1.5
    x0, ids0, t0, _, _ = make(4, 1, V, K, rest, odd=False)
    cols = np.concatenate([ids0[0][:5], np.arange(0, V, 60)])
    N = 2 * len(cols) + 1
    x = np.repeat(x0, N, 0)
    x = np.round(x * 64) / 64  # steps are exact
    for i, v in enumerate(cols):
        x[2 * i, v] += h
        x[2 * i + 1, v] -= h
    x = x.astype(np.float32)
    ids, t = np.repeat(ids0, N, 0), np.repeat(t0, N, 0)
    n, w = np.full(N, K, np.int32), np.ones(N, np.float32)
    loss, grad = run(torch, pz, x, ids, t, n, w, T, rest, torch.float32)
    d = max(distill_row(x[i], ids[i], t[i], T, rest)[2] for i in range(N))
    for i, v in enumerate(cols):
        slope = (float(loss[2 * i]) - float(loss[2 * i + 1])) / (2 * h)
        assert abs(slope - grad[N - 1, v]) <= h * h / 6 / T + (d + 2.0 ** -23) / h, (v, slope, grad[N - 1, v])


def test_autograd(cuda, pz):
    """distill_loss: the same gradients as the calls, upstream gradients that
    are expanded, logits used twice, and a second backward refused."""
    torch = cuda
    N, V, K = 9, 3001, 12
    x, ids, t, n, w = make(2, N, V, K, True)
    ids_d, t_d, n_d, w_d = (torch.from_numpy(a).cuda() for a in (ids, t, n, w))
    for dtype, half in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
        xb = x if dtype is torch.float32 else bf16_round(x)
        leaf = torch.from_numpy(xb).cuda().to(dtype).requires_grad_(True)
        kw = dict(weight=w_d, temperature=1.0, mode=pz.DISTILL_REST, n_list=n_d)
        loss = pz.distill_loss(leaf, ids_d, t_d, **kw)
        loss.sum().backward()  # the upstream gradient is one expanded number
        check(xb, ids, t, n, w, 1.0, True, loss.detach().cpu().numpy(), leaf.grad.float().cpu().numpy(), half)
        one = leaf.grad.clone()
        again = pz.distill_loss(leaf, ids_d, t_d, **kw).sum() * 2 + pz.distill_loss(leaf, ids_d, t_d, **kw).sum()
        leaf.grad = None
        again.backward()
        assert torch.allclose(leaf.grad.float(), 3 * one.float(), rtol=4 * half + 1e-6, atol=1e-12)
        wide = torch.zeros(N, V + 3, device="cuda", dtype=dtype)
        wide[:, :V] = leaf.detach()
        wide.requires_grad_(True)
        pz.distill_loss(wide[:, :V], ids_d, t_d, **kw).sum().backward()  # rows apart from one another
        # (a row's sums are grouped by its 16-byte vectors: other bits, the same bounds)
        check(xb, ids, t, n, w, 1.0, True, loss.detach().cpu().numpy(), wide.grad[:, :V].float().cpu().numpy(), half)
        assert not wide.grad[:, V:].any()
        leaf2 = leaf.detach().clone().requires_grad_(True)
        loss = pz.distill_loss(leaf2 * 1, ids_d, t_d, **kw).sum()
        g, = torch.autograd.grad(loss, leaf2, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_same_bits_each_time_and_in_a_graph(cuda, pz):
    torch = cuda
    N, V, K = 40, 50001, 33
    x, ids, t, n, w = make(6, N, V, K, True)
    dev = [torch.from_numpy(a).cuda() for a in (x, ids, t, n, w)]
    kw = dict(weight=dev[4], mode=pz.DISTILL_REST, n_list=dev[3])
    loss, grad = torch.empty(N, device="cuda"), torch.empty(N, V, device="cuda")
    pz.distill_loss_grad(dev[0], dev[1], dev[2], loss, grad, **kw)
    l0, g0 = loss.clone(), grad.clone()
    g = torch.cuda.CUDAGraph()
    stats = torch.empty(N, 4, device="cuda")
    grad2, loss2 = torch.empty_like(grad), torch.empty_like(loss)
    with torch.cuda.graph(g):
        pz.distill_loss_grad(dev[0], dev[1], dev[2], loss, grad, **kw)
        pz.distill_forward(dev[0], dev[1], dev[2], loss2, stats, **kw)
        pz.distill_backward(dev[0], dev[1], dev[2], stats, grad2, **kw)
    for _ in range(3):
        loss.zero_(), grad.zero_(), loss2.zero_(), grad2.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, l0) and torch.equal(grad, g0) and torch.equal(loss2, l0)
        assert torch.allclose(grad2, g0, rtol=1e-6, atol=1e-12)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [(torch.empty_like(loss), torch.empty_like(grad)) for _ in range(4)]
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(outs):
        pz.distill_loss_grad(dev[0], dev[1], dev[2], a, b, stream=(s1, s2)[i % 2], **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(a, l0) and torch.equal(b, g0) for a, b in outs)


def test_autograd_on_streams_and_in_a_graph(cuda, pz):
    """The differentiable form on a stream that is not the current one's, and
    forward and backward captured together."""
    torch = cuda
    N, V, K = 12, 20003, 10
    x, ids, t, n, w = make(14, N, V, K, False)
    ids_d, t_d, n_d, w_d = (torch.from_numpy(a).cuda() for a in (ids, t, n, w))
    kw = dict(weight=w_d, temperature=2.0, n_list=n_d)

    def both(leaf):
        loss = pz.distill_loss(leaf, ids_d, t_d, **kw)
        return loss.detach(), torch.autograd.grad(loss.sum(), leaf)[0]

    leaf = torch.from_numpy(x).cuda().requires_grad_(True)
    want = both(leaf)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = both(leaf)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    del got
    static = torch.zeros(N, V, device="cuda").requires_grad_(True)
    with torch.cuda.stream(side):
        both(static)  # warm-up, as a user captures
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both(static)
    for scale in (1.0, 0.5):
        with torch.no_grad():
            static.copy_(leaf.detach() * scale)
        g.replay()
        torch.cuda.synchronize()
        ref = both((leaf.detach() * scale).requires_grad_(True))
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


def test_offsets_past_32_bits(cuda, pz):
    torch = cuda
    N, V, K, ld = 3, 5000, 9, (1 << 30) + 8
    x, ids, t, n, w = make(12, N, V, K, False, odd=False)
    x = bf16_round(x)
    buf = torch.zeros(2 * ld + V, dtype=torch.bfloat16, device="cuda")
    view = buf.as_strided((N, V), (ld, 1))
    view.copy_(torch.from_numpy(x).cuda())
    loss = torch.empty(N, device="cuda")
    dev = [torch.from_numpy(a).cuda() for a in (ids, t, w)]
    pz.distill_loss_grad(view, dev[0], dev[1], loss, view, weight=dev[2])
    check(x, ids, t, n, w, 1.0, False, loss.cpu().numpy(), view.float().cpu().numpy(), 2.0 ** -8)


def test_from_the_samplers_lists(cuda, pz):
    """A teacher's batch through the sampler with its list outputs, then the
    student's loss against those lists: the path in use."""
    torch = cuda
    N, V, K = 24, 32000, 20
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    teacher = torch.randn(N, V, generator=g, device="cuda") * 3
    student = (teacher + torch.randn(N, V, generator=g, device="cuda")).requires_grad_(True)
    s = pz.Sampler(0, max_batch=N, max_vocab=V, max_top_k=32, max_history=0)
    cfg = pz.configs_to_device(pz.make_configs(N, temperature=1.0, top_k=K, top_p=1.0))
    rng = torch.arange(1, N + 1, dtype=torch.int64, device="cuda")
    tok = torch.empty(N, dtype=torch.int32, device="cuda")
    ids = torch.empty(N, 32, dtype=torch.int32, device="cuda")
    lp = torch.empty(N, 32, device="cuda")
    n = torch.empty(N, dtype=torch.int32, device="cuda")
    s.sample(teacher, cfg, rng, tok, max_top_k=32, no_full_vocab=True, cand_ids=ids, n_cand=n, cand_logprobs=lp)
    loss = pz.distill_loss(student, ids, lp, n_list=n, mode=pz.DISTILL_REST)
    loss.mean().backward()
    torch.cuda.synchronize()
    s.close()
    assert bool((n == K).all())
    check(student.detach().cpu().numpy(), ids.cpu().numpy(), lp.cpu().numpy(), n.cpu().numpy(),
          np.full(N, 1.0, np.float32), 1.0, True, loss.detach().cpu().numpy(), student.grad.cpu().numpy() * N,
          2.0 ** -22)
    # the lists are the teacher's own top ids and log-probabilities (1e-4, as the sampler promises)
    want = torch.log_softmax(teacher.double(), 1)
    top = want.topk(K, 1)
    assert torch.equal(top.indices.int(), ids[:, :K]) and float((top.values - lp[:, :K]).abs().max()) < 1e-4


def test_wrapper_refuses(cuda, pz):
    torch = cuda
    x = torch.zeros(4, 100, device="cuda")
    ids = torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    t = torch.zeros(4, 3, device="cuda")
    loss = torch.empty(4, device="cuda")
    with pytest.raises(TypeError):
        pz.distill_forward(x, ids.long(), t, loss)
    with pytest.raises(ValueError):
        pz.distill_forward(x, ids[:3], t[:3], loss)
    with pytest.raises(ValueError):
        pz.distill_forward(x, ids, t, loss[:3])
    with pytest.raises(pz.PZError):
        pz.distill_forward(x, ids, t, loss, temperature=0.0)
    with pytest.raises(pz.PZError):
        pz.distill_forward(x, ids, t, loss, mode=5)
    with pytest.raises(pz.PZError):
        pz.distill_forward(x, ids[:, :0], t[:, :0], loss)
    with pytest.raises(ValueError):
        pz.distill_loss_grad(x, ids, t, loss, torch.zeros(4, 99, device="cuda"))
    big = torch.zeros(9, 100, device="cuda")
    with pytest.raises(pz.PZError):
        pz.distill_loss_grad(big[:4], ids, t, loss, big[1:5])
    assert pz.distill_loss(x[:0], ids[:0], t[:0]).shape == (0,)


@pytest.mark.parametrize("T", [0.5, 0.01, 1e-3])
def test_list_values_keep_their_differences_at_any_temperature(cuda, pz, T):
    """Only the differences of a list's values count: values at the type's
    lowest (which a division by T < 1 takes to -inf), far from zero beside
    their differences (which it rounds away), and at either end of the type."""
    torch = cuda
    N, V, K = 8, 3000, 12
    x, ids, t, n, w = make(41, N, V, K, False, odd=False)
    x *= np.float32(T)                            # student and teacher in units of T
    t *= np.float32(T)
    t[0] = LOWEST                                 # a flat list
    t[1, 3:] = LOWEST                             # padded with the lowest value
    t[2] -= np.float32(20.0)                      # (rounded here: the oracle sees the same values)
    t[3] += np.float32(1000.0)
    t[4] = -LOWEST
    t[5], t[5, 4] = LOWEST, -LOWEST               # one id takes it all
    t[6, ::2] = -np.inf
    for how in ("both", "one"):
        loss, grad = run(torch, pz, x, ids, t, n, w, T, False, torch.float32, how=how)
        check(x, ids, t, n, w, T, False, loss, grad, 2.0 ** -24)
        assert np.isfinite(loss).all() and (loss != 0).all()


def test_a_student_masked_off_the_list(cuda, pz):
    """Every id off the list is -inf: REST holds what the list leaves against
    nothing (loss +inf, a gradient on the list alone), LIST is finite."""
    torch = cuda
    N, V, K = 4, 4001, 9
    x, ids, t, n, w = make(51, N, V, K, True, odd=False)
    on = np.zeros((N, V), dtype=bool)
    np.put_along_axis(on, ids, True, 1)
    x[~on] = -np.inf
    for rest in (True, False):
        for how in ("both", "one"):
            loss, grad = run(torch, pz, x, ids, t, n, w, 1.0, rest, torch.float32, how=how)
            check(x, ids, t, n, w, 1.0, rest, loss, grad, 2.0 ** -24)
            assert (loss == np.inf).all() == rest and np.isfinite(grad).all() and not grad[~on].any()
