"""The LM head in 8-bit integers (pz_quantize_rows_i8, pz_matmul_i8,
pz_lm_head_logits_i8) against numpy: quantisation and integer sums exactly,
products within their three fp32 roundings of fp64."""
import numpy as np
import pytest

from rows_ref import bf16_round

pytestmark = pytest.mark.gpu

F32 = np.float32


def quantize_ref(x):
    """(q, scale) of float32 rows by the definition's fp32 steps."""
    with np.errstate(all="ignore"):
        top = np.abs(x).max(1)
        bad = ~np.isfinite(x).all(1)
        some = ~bad & (top >= F32(2.0 ** -100))
        inv = np.where(some, F32(127) / top, F32(0)).astype(F32)
        scale = np.where(bad, F32(np.nan), np.where(some, top / F32(127), F32(0))).astype(F32)
        q = np.where(some[:, None], np.rint(x * inv[:, None]), 0)
    return q.astype(np.int8), scale


def padded(torch, rows, cols, extra=0, fill=99):
    ld = (cols + 15) // 16 * 16 + extra
    buf = torch.full((rows + 1, ld), fill, dtype=torch.int8, device="cuda")
    return buf, buf[:rows, :cols]


def product_ref(q, s, w, ws):
    acc = q.astype(np.float64) @ w.astype(np.float64).T  # exact: below 2^53
    return acc * s.astype(np.float64)[:, None] * ws.astype(np.float64)[None, :]


def check_product(got, want, bf16):
    """int -> fp32, the scales' product and the product: 3 half steps of fp32;
    bf16 output: one more of 2^-8."""
    rel = 3.1 * 2.0 ** -24 + (2.0 ** -8 if bf16 else 0.0)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = np.isnan(want) | (np.abs(got.astype(np.float64) - want) <= rel * np.abs(want) + 1e-44)
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 0), (3, 7, 1), (5, 100, 3), (9, 2560, 0), (4, 4099, 1), (7, 9000, 0),
                                   (300, 16, 0), (2, 131071, 1)], ids=str)
def test_rows_are_quantised(cuda, pz, shape, dtype):
    torch = cuda
    rows, cols, gap = shape
    r = np.random.default_rng(cols)
    x = (r.standard_normal((rows, cols)) * np.exp(r.standard_normal((rows, 1)) * 5)).astype(F32)
    if rows >= 5:
        x[0] = 0
        x[1] *= F32(1e-33)                      # below 2^-100
        x[2, cols // 2] = np.inf
        x[3, 0] = np.nan
        x[4, cols - 1] = 3e38                   # the others become 0
    if dtype == "bf16":
        x = bf16_round(x)
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    xs = torch.full((rows, cols + gap), 5.0, dtype=td, device="cuda")[:, :cols]
    xs.copy_(torch.from_numpy(x).cuda())
    buf, q = padded(torch, rows, cols, 16)
    scale = torch.full((rows + 1,), -9.0, device="cuda")
    pz.quantize_rows_i8(xs, q, scale)
    torch.cuda.synchronize()
    want_q, want_s = quantize_ref(x)
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert np.array_equal(scale[:rows].cpu().numpy(), want_s, equal_nan=True) and float(scale[rows]) == -9
    assert bool((buf[:rows, cols:] == 99).all()) and bool((buf[rows] == 99).all())


def tie_rows(rows, cols):
    """float32 rows whose values lie on either side of the steps' middles: the
    product in fp32 is a middle where the unrounded one is a little off it."""
    r = np.random.default_rng(cols)
    top = (1 + r.random((rows, 1))).astype(F32)
    inv = (F32(127) / top).astype(F32)
    x = ((r.integers(-127, 127, (rows, cols)) + 0.5) / inv.astype(np.float64)).astype(F32)
    for _ in range(2):
        x = np.where(r.random(x.shape) < 0.3, np.nextafter(x, r.choice([F32(-4), F32(4)], x.shape)), x).astype(F32)
    x = np.clip(x, -top, top)
    x[:, 0] = top[:, 0]
    return x, inv


@pytest.mark.parametrize("gap", [0, 1])
@pytest.mark.parametrize("cols", [1000, 4096, 5001])
def test_products_are_rounded_before_the_whole_number_is_taken(cuda, pz, cols, gap):
    torch = cuda
    x, inv = tie_rows(8, cols)
    want = quantize_ref(x)[0]
    assert (np.rint(x.astype(np.float64) * inv.astype(np.float64)) != want).sum() > 20   # one rounding moves them
    xs = torch.zeros(8, cols + gap, device="cuda")[:, :cols]
    xs.copy_(torch.from_numpy(x).cuda())
    buf, q = padded(torch, 8, cols)
    scale = torch.empty(8, device="cuda")
    pz.quantize_rows_i8(xs, q, scale)
    assert np.array_equal(q.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [9, 2051, 4103, 9001])
def test_infinities_and_nan_at_either_end_of_a_row(cuda, pz, cols, dtype):
    torch = cuda
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    xs = torch.ones(5, cols, dtype=td, device="cuda")      # odd: every row at another alignment
    bad = [(0, 0, np.nan), (1, cols - 1, np.nan), (2, 0, -np.inf), (3, cols - 1, np.inf)]
    for row, col, v in bad:
        xs[row, col] = float(v)
    buf, q = padded(torch, 5, cols)
    scale = torch.empty(5, device="cuda")
    pz.quantize_rows_i8(xs, q, scale)
    assert scale[:4].isnan().all() and (q[:4] == 0).all()
    assert scale[4].item() == F32(1) / F32(127) and (q[4] == 127).all()


SHAPES = [
    # M, N, K
    (1, 1, 1), (1, 130, 33), (2, 127, 128), (3, 129, 16), (15, 300, 100), (16, 128, 256), (17, 1000, 129),
    (33, 500, 640), (64, 257, 1000), (100, 700, 4096), (129, 333, 200), (255, 129, 96), (256, 640, 512),
    (257, 1001, 300), (300, 19000, 64), (64, 257, 40), (65, 1, 16), (70, 255, 1), (513, 3, 131), (1000, 257, 700), (513, 400, 2560), (1, 40000, 512), (8, 32003, 131),
]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_products(cuda, pz, shape, out):
    torch = cuda
    M, N, K = shape
    r = np.random.default_rng(M * 7 + N + K)
    qa = r.integers(-128, 128, (M, K)).astype(np.int8)
    qw = r.integers(-128, 128, (N, K)).astype(np.int8)
    sa = (0.5 + r.random(M)).astype(F32)
    sw = (1e-3 + 1e-2 * r.random(N)).astype(F32)
    if M > 2:
        sa[1] = 0
        sa[2] = np.nan
    abuf, a = padded(torch, M, K, 32)
    wbuf, w = padded(torch, N, K)
    a.copy_(torch.from_numpy(qa))
    w.copy_(torch.from_numpy(qw))
    td = torch.float32 if out == "f32" else torch.bfloat16
    obuf = torch.full((M + 1, N + 3), 7.0, dtype=td, device="cuda")
    o = obuf[:M, :N]
    pz.matmul_i8(a, torch.from_numpy(sa).cuda(), w, torch.from_numpy(sw).cuda(), o)
    torch.cuda.synchronize()
    check_product(o.float().cpu().numpy(), product_ref(qa, sa, qw, sw), out == "bf16")
    assert bool((obuf[:M, N:] == 7).all()) and bool((obuf[M] == 7).all())


def test_sums_of_the_largest_values(cuda, pz):
    """|sum| up to 2^31 - 2^14: the integers neither wrap nor saturate."""
    torch = cuda
    M, N, K = 3, 200, 131071
    a = torch.full((M, (K + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((N, (K + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :K]
    w[1::2] = 127
    one = torch.ones(256, device="cuda")
    out = torch.empty(M, N, device="cuda")
    pz.matmul_i8(a, one, w, one, out)
    assert bool((out[:, 0::2] == float(F32(K * 16384))).all()) and bool((out[:, 1::2] == float(F32(-K * 16256))).all())


@pytest.mark.parametrize("hidden", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 2560, 32000), (5, 1000, 3001), (70, 4096, 2000), (260, 513, 4000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_head(cuda, pz, shape, hidden):
    """Weights quantised by the library, tokens on the fly; against the
    definition, and against the unquantised product within the quantisation
    errors (half a step of each factor)."""
    torch = cuda
    B, dim, V = shape
    r = np.random.default_rng(dim)
    x = r.standard_normal((B, dim)).astype(F32)
    if hidden == "bf16":
        x = bf16_round(x)
    w = (r.standard_normal((V, dim)) * 0.05).astype(F32)
    _, wq = padded(torch, V, dim)
    ws = torch.empty(V, device="cuda")
    pz.quantize_rows_i8(torch.from_numpy(w).cuda(), wq, ws)
    _, hq = padded(torch, B, dim)
    hs = torch.empty(B, device="cuda")
    h = torch.from_numpy(x).cuda().to(torch.float32 if hidden == "f32" else torch.bfloat16)
    logits = torch.empty(B, V, device="cuda")
    pz.lm_head_i8(h, wq, ws, logits, hq, hs)
    torch.cuda.synchronize()
    (q, s), (qw, sw) = quantize_ref(x), quantize_ref(w)
    got = logits.cpu().numpy()
    check_product(got, product_ref(q, s, qw, sw), False)
    full = x.astype(np.float64) @ w.astype(np.float64).T
    step = (s.astype(np.float64) / 2)[:, None] * np.abs(w).sum(1)[None, :] + (
        np.abs(x).sum(1) + dim * s / 2)[:, None] * (sw.astype(np.float64) / 2)[None, :]
    assert np.all(np.abs(got - full) <= step * (1 + 1e-5) + 1e-6)
    # the unaligned and the bf16 output
    wide = torch.full((B, V + 1), 3.0, device="cuda", dtype=torch.bfloat16)
    pz.lm_head_i8(h, wq, ws, wide[:, 1:], hq, hs)
    torch.cuda.synchronize()
    assert torch.equal(wide[:, 1:], logits.to(torch.bfloat16)) and bool((wide[:, 0] == 3).all())


def test_rows_past_32_bits(cuda, pz):
    """Weights and logits whose last elements lie past 2^31."""
    torch = cuda
    V, dim, B = 70001, 64, 3
    ld = 32768
    buf = torch.zeros((V - 1) * ld + dim, dtype=torch.int8, device="cuda")
    w = buf.as_strided((V, dim), (ld, 1))
    w.copy_(torch.randint(-127, 128, (V, dim), device="cuda", dtype=torch.int8))
    a = torch.randint(-127, 128, (B, dim), device="cuda", dtype=torch.int8)
    ones = torch.ones(V, device="cuda")
    ld_o = (1 << 30) + 4
    obuf = torch.zeros(2 * ld_o + V, dtype=torch.bfloat16, device="cuda")
    out = obuf.as_strided((B, V), (ld_o, 1))
    pz.matmul_i8(a, ones, w, ones, out)
    want = (a.double() @ w.double().T).to(torch.bfloat16)
    assert torch.equal(out, want)


def test_graph_and_two_streams(cuda, pz):
    torch = cuda
    B, dim, V = 20, 640, 9000
    _, wq = padded(torch, V, dim)
    wq.random_(-127, 128)
    ws = torch.rand(V, device="cuda")
    hs = [torch.randn(B, dim, device="cuda") for _ in range(4)]
    bufs = [(padded(torch, B, dim)[1], torch.empty(B, device="cuda"), torch.empty(B, V, device="cuda")) for _ in hs]
    want = []
    for h, (q, s, o) in zip(hs, bufs):
        pz.lm_head_i8(h, wq, ws, o, q, s)
        want.append(o.clone())
        o.zero_()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i, (h, (q, s, o)) in enumerate(zip(hs, bufs)):
        pz.lm_head_i8(h, wq, ws, o, q, s, stream=(s1, s2)[i % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for (_, _, o), w in zip(bufs, want))
    x = hs[0].clone()
    q, s, o = bufs[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pz.lm_head_i8(x, wq, ws, o, q, s)
    for i in (1, 2, 0):
        x.copy_(hs[i])  # a replay reads what is there then
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[i])


def test_head_rules_sampler_and_distillation_together(cuda, pz):
    """A decode step and a training step as they are used: the 8-bit head
    makes the logits, a grammar and biases constrain them, the sampler draws
    and lists, and the student (the same head's dequantised weights, trained
    in fp32) learns from the lists."""
    torch = cuda
    B, dim, V, K = 12, 256, 8000, 16
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    w = torch.randn(V, dim, generator=gen, device="cuda") * 0.2
    h = torch.randn(B, dim, generator=gen, device="cuda")
    _, wq = padded(torch, V, dim)
    ws = torch.empty(V, device="cuda")
    pz.quantize_rows_i8(w, wq, ws)
    _, hq = padded(torch, B, dim)
    hs = torch.empty(B, device="cuda")
    logits = torch.empty(B, V, device="cuda")
    allowed = torch.zeros(1, V, dtype=torch.bool, device="cuda")
    allowed[0, 5::7] = True
    words = (allowed.view(1, -1, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
    index = torch.zeros(B, dtype=torch.int32, device="cuda")
    index[::2] = -1
    ban = torch.tensor([12, 5], dtype=torch.int32, device="cuda")
    off = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    off[3:] = 2  # row 2 is biased
    cfg = pz.configs_to_device(pz.make_configs(B, temperature=1.0, top_k=K, top_p=1.0))
    rng = torch.arange(1, B + 1, dtype=torch.int64, device="cuda")
    tok, n = (torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(2))
    ids = torch.empty(B, K, dtype=torch.int32, device="cuda")
    lp = torch.empty(B, K, device="cuda")
    s = pz.Sampler(0, max_batch=B, max_vocab=V, max_top_k=K, max_history=0)

    def step():
        pz.lm_head_i8(h, wq, ws, logits, hq, hs)
        pz.process_logits(logits, mask=mask, mask_index=index, bias_ids=ban,
                          bias_vals=torch.full((2,), float("-inf"), device="cuda"), bias_off=off)
        s.sample(logits, cfg, rng, tok, max_top_k=K, no_full_vocab=True, cand_ids=ids, n_cand=n, cand_logprobs=lp)

    step()
    torch.cuda.synchronize()
    s.close()
    assert bool((tok[1::2] % 7 == 5).all()) and bool((ids[1::2] % 7 == 5).all()) and bool((n == K).all())
    assert not bool(((ids[2] == 12) | (ids[2] == 5)).any())
    deq = wq.float() * ws[:, None]
    full = (hq.float() * hs[:, None]).double() @ deq.double().T
    full[1::2] = full[1::2].masked_fill(~allowed, float("-inf"))
    full[2, ban.long()] = float("-inf")
    want = torch.log_softmax(full, 1).gather(1, ids.long())
    assert float((want - lp).abs().max()) < 1e-4  # the sampler's own bound on log-probabilities
    weights = deq.clone().requires_grad_(True)
    student = h @ weights.T
    loss = pz.distill_loss(student, ids, lp, n_list=n, mode=pz.DISTILL_REST)
    loss.sum().backward()
    p = lp.double().exp()
    rho = (1 - p.sum(1)).clamp(min=0)
    x = student.detach().double()
    on = torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids.long(), True)
    q = torch.softmax(x, 1)
    g = q * (p.sum(1) + rho)[:, None] - torch.zeros_like(x).scatter_(1, ids.long(), p) - rho[:, None] * torch.softmax(
        x.masked_fill(on, float("-inf")), 1)
    want = g.T @ h.double()
    got = weights.grad.double()
    # fp32 products of B terms of the gradient's own error (1e-5 of its parts)
    bound = 2e-5 * ((q + on + rho[:, None]).T @ h.double().abs()) + 1e-9
    assert bool(((got - want).abs() <= bound).all())


def test_wrapper_refuses(cuda, pz):
    torch = cuda
    _, w = padded(torch, 50, 40)
    s = torch.ones(50, device="cuda")
    h = torch.zeros(4, 40, device="cuda")
    _, q = padded(torch, 4, 40)
    out = torch.empty(4, 50, device="cuda")
    with pytest.raises(pz.PZError):  # rows 40 bytes apart
        pz.lm_head_i8(h, torch.zeros(50, 40, dtype=torch.int8, device="cuda"), s, out, q, s)
    with pytest.raises(ValueError):
        pz.lm_head_i8(h, w, s, out[:, :49], q, s)
    with pytest.raises(ValueError):
        pz.lm_head_i8(h, w, s[:49], out, q, s)
    with pytest.raises(ValueError):
        pz.lm_head_i8(h, w.float(), s, out, q, s)
    with pytest.raises(TypeError):
        pz.lm_head_i8(h.half(), w, s, out, q, s)
    with pytest.raises(TypeError):
        pz.matmul_i8(q, s, w, s, out.half())
    with pytest.raises(ValueError):
        pz.quantize_rows_i8(h, q[:3], s)
    pz.lm_head_i8(h[:0], w, s, out[:0], q[:0], s)
