"""pz_process_logits on batches of many waves of CTAs: parts of several whole
batches of vectors, the fewer list threads of such batches, and lists with
more ids in a part than its table takes.  Bit for bit against numpy's fp32
steps, like the small batches of test_gpu_rules.py."""
import numpy as np
import pytest

from rows_ref import bf16_round, pack_mask, process_row

pytestmark = pytest.mark.gpu

B = 640


def make(torch, V, seed, lists, masks):
    """Logits on the device, rules as numpy arrays.  Rows 1 and 2 of every 40
    have thousands of distinct ids next to one another (and twice over), row 3
    one id only, row 4 nothing."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(B, V, generator=g, device="cuda") * 4
    r = np.random.default_rng(seed)
    d = dict(x=x, V=V, cfg=None, hist=None, bias=None, allowed=None, index=None)
    if lists:
        d["cfg"] = np.stack([r.choice([1.0, 1.1, 1.3, 0.8], B), r.choice([0.0, 0.2, 0.5], B),
                             r.choice([0.0, 0.1], B)], 1).astype(np.float32)
        hist, bias = [], []
        for b in range(B):
            kind = b % 40
            if kind in (1, 2):
                n = (3000, min(16000, V))[kind - 1]
                at = r.integers(0, V - n + 1)
                h = r.permutation(np.arange(at, at + n))
                h = np.concatenate([h, r.choice(h, n // 3), [-1, V, V + 7]])
                t = np.concatenate([np.arange(at, at + n, 2), np.arange(at, at + n, 6)[::-1], [-5, V]])
            elif kind == 3:
                h, t = np.full(500, V - 1), np.full(40, V // 2)
            elif kind == 4:
                h = t = np.zeros(0)
            else:
                h, t = r.integers(-3, V + 3, r.integers(0, 900)), r.integers(-2, V + 2, r.integers(0, 60))
            hist.append(h.astype(np.int32))
            bias.append((t.astype(np.int32), (r.standard_normal(len(t)) * 9).astype(np.float32)))
        d["hist"], d["bias"] = hist, bias
    if masks:
        d["allowed"] = r.random((7, V)) < np.array([0.5, 0.02, 0.98, 0.0, 1.0, 0.9995, 0.0005])[:, None]
        d["index"] = r.integers(-1, 8, B).astype(np.int32)  # 7 is past the end: no mask
        d["index"][1::40] = 0
        d["index"][2::40] = 2
    return d


def rules(torch, pz, d):
    kw = {}
    if d["hist"] is not None:
        kw["cfg"] = pz.configs_to_device(pz.make_configs(B, rep=d["cfg"][:, 0], freq=d["cfg"][:, 1], pres=d["cfg"][:, 2]))

        def csr(lists):
            off = np.cumsum([0] + [len(v) for v in lists]).astype(np.int32)
            return torch.from_numpy(np.concatenate(lists)).cuda(), torch.from_numpy(off).cuda()
        kw["hist"], kw["hist_off"] = csr(d["hist"])
        kw["bias_ids"], kw["bias_off"] = csr([i for i, _ in d["bias"]])
        kw["bias_vals"], _ = csr([v for _, v in d["bias"]])
    if d["allowed"] is not None:
        kw["mask"] = torch.from_numpy(pack_mask(d["allowed"], (d["V"] + 31) // 32 + 1)).cuda()
        kw["mask_index"] = torch.from_numpy(d["index"]).cuda()
    return kw


def placed(torch, x, dtype, ld, lead):
    """x in a buffer of 7s: rows ld apart, `lead` elements in front, a row
    behind.  (buffer, view)"""
    V = x.shape[1]
    buf = torch.full((lead + (B + 1) * ld,), 7.0, dtype=dtype, device="cuda")
    view = buf[lead:lead + B * ld].view(B, ld)[:, :V]
    view.copy_(x)
    return buf, view


@pytest.mark.parametrize("rule", ["masks", "lists", "lists_masks"])
@pytest.mark.parametrize("where", ["apart", "apart_odd", "in_place", "in_place_odd"])
@pytest.mark.parametrize("types", ["f32", "bf16", "bf16_f32"])
@pytest.mark.parametrize("V", [20011, 32768, 33003])
def test_large_batches(cuda, pz, V, types, where, rule):
    torch = cuda
    inplace, odd = where.startswith("in_place"), where.endswith("odd")
    if inplace and types == "bf16_f32":
        pytest.skip("a wider output is another buffer")
    d = make(torch, V, V + len(rule), "lists" in rule, "masks" in rule)
    ti = torch.float32 if types == "f32" else torch.bfloat16
    to = torch.bfloat16 if types == "bf16" else torch.float32
    ld = V + 3 if odd else (V + 7) // 8 * 8
    buf, x = placed(torch, d["x"], ti, ld, 1 if odd else 0)
    given = x.clone()
    obuf, out = (buf, x) if inplace else placed(torch, torch.zeros_like(d["x"]), to, ld, 3 if odd else 0)
    n = torch.full((B + 1,), -9, dtype=torch.int32, device="cuda")
    pz.process_logits(x, None if inplace else out, n_allowed=n, **rules(torch, pz, d))
    torch.cuda.synchronize()
    if not inplace:
        assert torch.equal(x, given)
    # all rows: what no rule names comes through as it is, what the mask takes is -inf
    named = torch.zeros(B, V, dtype=torch.bool)
    if d["hist"] is not None:
        for b in range(B):
            for ids in (d["hist"][b], d["bias"][b][0]):
                named[b, torch.from_numpy(ids[(ids >= 0) & (ids < V)]).long()] = True
    named = named.cuda()
    want = given.to(to)
    left = np.full(B, V)
    if d["allowed"] is not None:
        index = torch.from_numpy(d["index"]).cuda().long()
        has = (index >= 0) & (index < 7)
        taken = ~torch.from_numpy(d["allowed"]).cuda()[index.clamp(0, 6)] & has[:, None]
        want = want.masked_fill(taken, float("-inf"))
        named &= ~taken
        left = V - taken.sum(1).cpu().numpy()
    assert bool(((out == want) | named).all())
    assert np.array_equal(n[:B].cpu().numpy(), left) and int(n[B]) == -9
    # some rows whole, those of the long lists among them
    for b in sorted(set(range(0, B, 59)) | {1, 2, 3, 4, 41, 42, B - 39, B - 38, B - 1}):
        k = -1 if d["index"] is None else int(d["index"][b])
        row = process_row(given[b].float().cpu().numpy(), V, None if d["cfg"] is None else d["cfg"][b],
                          None if d["hist"] is None else d["hist"][b], None if d["bias"] is None else d["bias"][b],
                          d["allowed"][k] if 0 <= k < 7 else None)
        row = bf16_round(row) if to is torch.bfloat16 else row
        assert np.array_equal(out[b].float().cpu().numpy(), row), b
    first = (1 if inplace else 3) if odd else 0
    rest = torch.ones(obuf.numel(), dtype=torch.bool, device="cuda")
    rest[first:first + B * ld].view(B, ld)[:, :V] = False
    assert bool((obuf[rest] == 7).all())


@pytest.mark.parametrize("inplace", [False, True], ids=["apart", "in_place"])
def test_lists_longer_than_a_table_in_a_small_batch(cuda, pz, inplace):
    """One wave of CTAs (the more list threads), a part of 128 vectors at
    least: 3 rows of 2^20 columns whose lists fill every part's table twice
    over."""
    torch = cuda
    rows, V = 3, 1 << 20
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn(rows, V, generator=g, device="cuda") * 4
    given = x.clone()
    r = np.random.default_rng(6)
    hist = [r.permutation(V)[:V // 2].astype(np.int32), np.arange(V, dtype=np.int32)[::-1].copy(),
            np.repeat(np.arange(100, 5100, dtype=np.int32), 3)]
    bias = [r.permutation(V)[:V // 3].astype(np.int32), np.arange(0, V, 3, dtype=np.int32), np.arange(3000, dtype=np.int32)]
    vals = [(r.standard_normal(len(b)) * 5).astype(np.float32) for b in bias]
    pen = np.array([[1.2, 0.3, 0.1], [0.9, 0.0, 0.2], [1.0, 0.25, 0.0]], dtype=np.float32)
    allowed = r.random((1, V)) < 0.6

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def off(lists):
        return dev(np.cumsum([0] + [len(v) for v in lists]).astype(np.int32))
    out = x if inplace else torch.empty_like(x)
    pz.process_logits(x, out, cfg=pz.configs_to_device(pz.make_configs(rows, rep=pen[:, 0], freq=pen[:, 1], pres=pen[:, 2])),
                      hist=dev(np.concatenate(hist)), hist_off=off(hist), bias_ids=dev(np.concatenate(bias)),
                      bias_vals=dev(np.concatenate(vals)), bias_off=off(bias), mask=dev(pack_mask(allowed, V // 32)),
                      mask_index=dev(np.array([0, -1, 0], dtype=np.int32)))
    for b in range(rows):
        want = process_row(given[b].cpu().numpy(), V, pen[b], hist[b], (bias[b], vals[b]), None if b == 1 else allowed[0])
        assert np.array_equal(out[b].cpu().numpy(), want), b
