"""pz_process_logits (penalties, biases, grammar masks on rows of logits)
against numpy: bit for bit against the contract's fp32 steps, and within
their roundings of fp64."""
import numpy as np
import pytest

from rows_ref import bf16_round, pack_mask, process_row

pytestmark = pytest.mark.gpu

SPECIALS = np.array([np.nan, np.inf, -np.inf, -np.finfo(np.float32).max, np.finfo(np.float32).max, 0.0, -0.0],
                    dtype=np.float32)


def make(seed, B, V, *, hist=True, bias=True, mask="own", specials=True):
    """Rows and their rules as numpy arrays: row 0 has empty lists, ids
    repeat and leave [0, V), one mask row allows nothing, one everything."""
    r = np.random.default_rng(seed)
    x = (r.standard_normal((B, V)) * 4).astype(np.float32)
    if specials and V > 8:
        for b in range(B):
            x[b, r.integers(0, V, 7)] = SPECIALS
    d = dict(x=x, B=B, V=V, cfg=None, hist=None, bias=None, allowed=None, index=None)
    if hist:
        d["cfg"] = np.stack([r.choice([1.0, 1.1, 1.3, 0.8], B), r.choice([0.0, 0.2, 0.5], B),
                             r.choice([0.0, 0.1], B)], 1).astype(np.float32)
        n = r.integers(0, 700, B)
        n[0] = 0
        d["hist"] = [np.where(r.random(k) < 0.5, r.integers(-3, V + 3, k), r.integers(0, min(V, 5), k)).astype(np.int32)
                     for k in n]
    if bias:
        n = r.integers(0, 40, B)
        n[0] = 0
        d["bias"] = [(r.integers(-2, min(V, 50) + 2, k).astype(np.int32), (r.standard_normal(k) * 9).astype(np.float32))
                     for k in n]
    if mask:
        rows = B if mask == "own" else 3
        d["allowed"] = r.random((rows, V)) < r.choice([0.02, 0.5, 0.98], (rows, 1))
        d["allowed"][0] = False
        if rows > 1:
            d["allowed"][1] = True
        if mask == "index":
            d["index"] = r.integers(-1, rows + 1, B).astype(np.int32)  # rows is past the end: no mask
    return d


def want_row(d, b, wide=False):
    allowed = None
    if d["allowed"] is not None:
        k = b if d["index"] is None else int(d["index"][b])
        allowed = d["allowed"][k] if 0 <= k < len(d["allowed"]) else None
    return process_row(d["x"][b], d["V"], None if d["cfg"] is None else d["cfg"][b],
                       None if d["hist"] is None else d["hist"][b], None if d["bias"] is None else d["bias"][b],
                       allowed, wide), int(d["V"] if allowed is None else allowed.sum())


def csr(torch, lists, dtype):
    off = np.cumsum([0] + [len(v) for v in lists]).astype(np.int32)
    flat = np.concatenate(lists).astype(dtype) if len(lists) else np.zeros(0, dtype)
    return torch.from_numpy(np.append(flat, flat[:0]).copy()).cuda(), torch.from_numpy(off).cuda()


def rules(torch, pz, d, words=None):
    kw = {}
    if d["hist"] is not None:
        c = pz.make_configs(d["B"], rep=d["cfg"][:, 0], freq=d["cfg"][:, 1], pres=d["cfg"][:, 2])
        kw["cfg"] = pz.configs_to_device(c)
        kw["hist"], kw["hist_off"] = csr(torch, d["hist"], np.int32)
    if d["bias"] is not None:
        kw["bias_ids"], kw["bias_off"] = csr(torch, [i for i, _ in d["bias"]], np.int32)
        kw["bias_vals"], _ = csr(torch, [v for _, v in d["bias"]], np.float32)
    if d["allowed"] is not None:
        words = words or (d["V"] + 31) // 32
        kw["mask"] = torch.from_numpy(pack_mask(d["allowed"], words)).cuda()
        if d["index"] is not None:
            kw["mask_index"] = torch.from_numpy(d["index"]).cuda()
    return kw


def strided(torch, x, dtype, ld, lead):
    """x in a buffer of 7s: rows ld apart, `lead` elements in front, one row
    of slack behind.  (buffer, view)"""
    B, V = x.shape
    buf = torch.full((lead + (B + 1) * ld,), 7.0, dtype=dtype, device="cuda")
    view = buf[lead:lead + B * ld].view(B, ld)[:, :V]
    view.copy_(torch.from_numpy(x).cuda().to(dtype))
    return buf, view


CASES = [
    # V, ld - V, lead elements, mask, lists
    (1, 0, 0, "own", True), (2, 1, 1, "own", True), (31, 0, 3, "index", True), (33, 2, 1, "own", True),
    (1000, 0, 0, None, True), (4095, 3, 5, "own", True), (4097, 0, 1, "index", True), (2048, 0, 0, "own", False),
    (20011, 5, 2, "own", True), (8192, 0, 0, "index", True),
]


@pytest.mark.parametrize("types", ["f32", "bf16", "bf16_f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("inplace", [False, True], ids=["apart", "in_place"])
def test_rows_match_the_contract(cuda, pz, case, types, inplace):
    torch = cuda
    if inplace and types == "bf16_f32":
        pytest.skip("a wider output is another buffer")
    V, gap, lead, mask, lists = case
    B = 6
    d = make(V * 31 + gap, B, V, hist=lists, bias=lists, mask=mask)
    ti = torch.float32 if types == "f32" else torch.bfloat16
    to = torch.bfloat16 if types == "bf16" else torch.float32
    if ti is torch.bfloat16:
        d["x"] = bf16_round(d["x"])
    buf, x = strided(torch, d["x"], ti, V + gap, lead)
    obuf, out = (buf, x) if inplace else strided(torch, np.zeros((B, V), np.float32), to, V + gap + 1, lead + 1)
    before = x.clone()
    n = torch.full((B + 1,), -9, dtype=torch.int32, device="cuda")
    pz.process_logits(x, None if inplace else out, n_allowed=n, **rules(torch, pz, d, (V + 31) // 32 + 2))
    torch.cuda.synchronize()
    got = out.float().cpu().numpy()
    for b in range(B):
        want, left = want_row(d, b)
        wide, _ = want_row(d, b, wide=True)
        if to is torch.bfloat16:
            want = bf16_round(want)
        assert np.array_equal(got[b], want, equal_nan=True), b
        # penalty: 4 roundings, bias 1, output 1 (of bf16: half a step of 2^-8)
        with np.errstate(all="ignore"):
            size = np.abs(wide) + np.abs(d["x"][b].astype(np.float64)) * 2 + 700 * 0.5 + 64
            off = np.abs(np.where(np.isfinite(wide) & np.isfinite(want), got[b] - wide, 0))
        half = 2.0 ** -8 if to is torch.bfloat16 else 2.0 ** -24
        assert np.all(off <= 6 * 2.0 ** -24 * np.where(np.isfinite(size), size, 3e38) + half * np.abs(
            np.where(np.isfinite(wide), wide, 0))), b
        assert int(n[b]) == left
    assert int(n[B]) == -9
    if not inplace:
        assert torch.equal(x.view(torch.int16 if ti is torch.bfloat16 else torch.int32),
                           before.view(torch.int16 if ti is torch.bfloat16 else torch.int32))
    # what lies between and behind the rows is as it was
    ld = out.stride(0)
    first = lead + (0 if inplace else 1)
    rest = torch.ones(obuf.numel(), dtype=torch.bool, device="cuda")
    rest[first:first + B * ld].view(B, ld)[:, :V] = False
    assert bool((obuf[rest] == 7).all())


def test_long_histories_and_large_rows(cuda, pz):
    """Histories longer than any context's, over rows of several tiles."""
    torch = cuda
    B, V = 3, 128256
    r = np.random.default_rng(5)
    d = make(9, B, V, specials=False)
    d["hist"] = [r.integers(0, V, 50000).astype(np.int32), np.full(70000, 4321, np.int32),
                 r.integers(0, 300, 9000).astype(np.int32)]
    x = torch.from_numpy(d["x"]).cuda()
    out = torch.empty_like(x)
    pz.process_logits(x, out, **rules(torch, pz, d))
    for b in range(B):
        assert np.array_equal(out[b].cpu().numpy(), want_row(d, b)[0]), b


def test_offsets_past_32_bits(cuda, pz):
    """The last row starts more than 2^31 elements into the buffer."""
    torch = cuda
    B, V, ld = 3, 5000, (1 << 30) + 8
    buf = torch.zeros(2 * ld + V, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((B, V), (ld, 1))
    d = make(11, B, V, specials=False)
    d["x"] = bf16_round(d["x"])
    x.copy_(torch.from_numpy(d["x"]).cuda())
    pz.process_logits(x, **rules(torch, pz, d))
    for b in range(B):
        assert np.array_equal(x[b].float().cpu().numpy(), bf16_round(want_row(d, b)[0])), b
    assert int(torch.count_nonzero(buf[V:ld])) == 0


def test_sampler_draws_the_same_from_processed_rows(cuda, pz, oracle_lib):
    """Penalties applied by process_logits and none in the sampler: the same
    tokens, lists and RNG words as the sampler's own penalties, f32 and bf16
    (widened to f32), and masked rows draw allowed ids only."""
    torch = cuda
    import cases
    from gpu_helpers import to_device
    for dtype in ("f32", "bf16"):
        spec = dict(seed=77, B=40, V=32000, sd=2.5, boosts=[8, 5.0, 15.0], hist_len=500, dtype=dtype,
                    cfg=dict(temperature=0.7, top_k=50, top_p=0.9, rep=1.2, freq=0.3, pres=0.1))
        x, cfg, rng, hist, off = to_device(torch, cases.build(spec))
        B, V = x.shape
        rng2 = rng.clone()
        a, b = (torch.full((B,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
        ia, ib = (torch.full((B, 64), -9, dtype=torch.int32, device="cuda") for _ in range(2))
        pa, pb = (torch.zeros(B, 64, device="cuda") for _ in range(2))
        s = pz.Sampler(0, max_batch=B, max_vocab=V, max_top_k=64, max_history=512)
        s.sample(x, cfg, rng, a, hist, off, max_top_k=64, no_full_vocab=True, cand_ids=ia, cand_probs=pa)
        y = torch.empty(B, V, device="cuda")
        pz.process_logits(x, y, cfg=cfg, hist=hist, hist_off=off)
        s.sample(y, cfg, rng2, b, max_top_k=64, no_full_vocab=True, cand_ids=ib, cand_probs=pb)
        assert torch.equal(a, b) and torch.equal(ia, ib) and torch.equal(pa, pb) and torch.equal(rng, rng2)
        # a grammar of 100 ids, in place, on the same stream
        allowed = np.zeros((1, V), dtype=bool)
        allowed[0, 7::320] = True
        mask = torch.from_numpy(pack_mask(allowed, V // 32)).cuda()
        n = torch.empty(B, dtype=torch.int32, device="cuda")
        pz.process_logits(y, mask=mask, mask_index=torch.zeros(B, dtype=torch.int32, device="cuda"), n_allowed=n)
        s.sample(y, cfg, rng2, b, max_top_k=64, no_full_vocab=True)
        assert bool((n == 100).all()) and bool((b % 320 == 7).all())
        s.close()


def test_graph_streams_and_two_calls_at_once(cuda, pz):
    torch = cuda
    B, V = 5, 9001
    d = make(21, B, V)
    kw = rules(torch, pz, d)
    x = torch.from_numpy(d["x"]).cuda()
    want = torch.from_numpy(np.stack([want_row(d, b)[0] for b in range(B)])).cuda()
    out = torch.zeros_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pz.process_logits(x, out, **kw)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(), want.nan_to_num())
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [torch.zeros_like(x) for _ in range(6)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        pz.process_logits(x, o, stream=(s1, s2)[i % 2], **kw)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.nan_to_num(), want.nan_to_num())


def test_other_device_is_not_the_current_one(cuda, pz):
    torch = cuda
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    x = torch.randn(4, 5000, device="cuda:1")
    y = torch.empty_like(x)
    pz.process_logits(x, y)
    torch.cuda.synchronize(1)
    assert torch.equal(x, y)


def test_wrapper_refuses(cuda, pz):
    torch = cuda
    x = torch.zeros(4, 100, device="cuda")
    m = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
    off = torch.zeros(5, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        pz.process_logits(x.t())
    with pytest.raises(ValueError):
        pz.process_logits(x, mask=m[:, :3])
    with pytest.raises(ValueError):
        pz.process_logits(x, torch.zeros(4, 99, device="cuda"))
    with pytest.raises(ValueError):
        pz.process_logits(x, bias_ids=off, bias_vals=x[0, :5], bias_off=off[:4])
    with pytest.raises(ValueError):
        pz.process_logits(x, hist=off.long(), hist_off=off)
    with pytest.raises(pz.PZError) as e:
        pz.process_logits(x, hist=off, hist_off=off)
    assert e.value.status == 1 and "cfg" in str(e.value)
    with pytest.raises(pz.PZError):
        pz.process_logits(x, mask=m[:3])
    with pytest.raises(TypeError):
        pz.process_logits(x.half())
    with pytest.raises(pz.PZError):  # the output overlaps the input
        big = torch.zeros(9, 100, device="cuda")
        pz.process_logits(big[:4], big[2:6])
    pz.process_logits(x[:0])  # an empty batch
    x.normal_()
    same = x.clone()
    pz.process_logits(x, hist=off[:0], hist_off=off, bias_ids=off[:0], bias_vals=x[0, :0], bias_off=off)
    assert torch.equal(x, same)  # lists without an entry
