"""pz_distill_* on batches of more rows than the GPU has CTA slots: one and
two CTAs a row, several whole batches of vectors each, streamed in the
backward pass.  Some rows against numpy in fp64 (rows_ref.distill_row), every
row's two gradients against one another."""
import numpy as np
import pytest

from rows_ref import close, distill_row

pytestmark = pytest.mark.gpu

V, K = 33003, 40


def make(torch, N, rest, dtype, ld, lead, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(N, V, generator=g, device="cuda") * 3
    j = torch.arange(K, device="cuda")
    first = torch.randint(0, V, (N, 1), generator=g, device="cuda")
    ids = (first + torch.randint(1, V // K, (N, 1), generator=g, device="cuda") * j) % V
    x.scatter_add_(1, ids, torch.rand(N, K, generator=g, device="cuda") * 6)
    t = torch.randn(N, K, generator=g, device="cuda") * 2
    n = torch.randint(1, K + 1, (N,), generator=g, device="cuda")
    n[::3] = K
    if rest:  # 2 to 40 % off the list
        t = torch.where(j[None] < n[:, None], t, float("-inf"))
        t = torch.log_softmax(t, 1) + torch.log1p(-(0.02 + 0.38 * torch.rand(N, 1, generator=g, device="cuda")))
    w = 0.5 + torch.rand(N, generator=g, device="cuda")
    w[5::17] = 0.0
    n[7::29] = 0
    x[5] = float("nan")  # padding may hold anything
    buf = torch.full((lead + (N + 1) * ld,), 7.0, dtype=dtype, device="cuda")
    view = buf[lead:lead + N * ld].view(N, ld)[:, :V]
    view.copy_(x)
    return buf, view, ids.int(), t, n.int(), w


@pytest.mark.parametrize("odd", [False, True], ids=["aligned", "odd"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rest", [False, True], ids=["list", "rest"])
@pytest.mark.parametrize("N", [1100, 1900])
def test_large_batches(cuda, pz, N, rest, dtype, odd):
    torch = cuda
    T = 1.0 if rest else 2.0
    td, half = (torch.float32, 2.0 ** -24) if dtype == "f32" else (torch.bfloat16, 2.0 ** -8)
    ld, lead = (V, 1) if odd else ((V + 7) // 8 * 8, 0)
    xbuf, x, ids, t, n, w = make(torch, N, rest, td, ld, lead, N + rest)
    kw = dict(weight=w, temperature=T, mode=pz.DISTILL_REST if rest else pz.DISTILL_LIST, n_list=n)
    loss, loss1 = (torch.full((N + 1,), -9.0, device="cuda") for _ in range(2))
    stats = torch.empty(N, 4, device="cuda")

    def out():
        buf = torch.full((lead + (N + 1) * ld,), 7.0, dtype=td, device="cuda")
        return buf, buf[lead:lead + N * ld].view(N, ld)[:, :V]
    gbuf, g = out()
    buf1, g1 = out()
    pz.distill_forward(x, ids, t, loss, stats, **kw)
    pz.distill_backward(x, ids, t, stats, g, **kw)
    pz.distill_loss_grad(x, ids, t, loss1, g1, **kw)
    # (of the same layout: a row's sums are grouped by its 16-byte vectors)
    inplace, inplace1 = (xbuf.clone()[lead:lead + N * ld].view(N, ld)[:, :V] for _ in range(2))
    pz.distill_backward(inplace, ids, t, stats, inplace, **kw)
    pz.distill_loss_grad(inplace1, ids, t, torch.empty(N, device="cuda"), inplace1, **kw)
    torch.cuda.synchronize()
    assert torch.equal(inplace, g) and torch.equal(inplace1, g1)
    for b in (gbuf, buf1):
        rest_of = torch.ones(b.numel(), dtype=torch.bool, device="cuda")
        rest_of[lead:lead + N * ld].view(N, ld)[:, :V] = False
        assert bool((b[rest_of] == 7).all())
    assert float(loss[N]) == float(loss1[N]) == -9
    none = (w == 0) | (n == 0)
    assert not bool(loss[:N][none].any()) and not bool(g[none].any()) and not bool(g1[none].any())
    # All rows: either gradient is within 2400 u (u = 2^-24) of the parts that
    # it is the difference of, mass q, p and rho e / S_off: an e is off by 141 u
    # at most here (65 units of its exponent), a sum by 442 u, one off the list
    # by 580 u, the pass's factor by 96 u, and rho by 36 u of a mass of 1, which
    # is 1800 u of the smallest rho of 0.02.
    for r in range(0, N, 128):
        s = slice(r, min(r + 128, N))
        xs, at = x[s].double() / T, ids[s].long()
        on = torch.arange(K, device="cuda")[None] < n[s][:, None]
        tt = t[s].double()
        p = (tt.exp() if rest else torch.softmax((tt / T).masked_fill(~on, float("-inf")), 1)).masked_fill(~on, 0)
        p = p.nan_to_num()
        parts = torch.softmax(xs, 1)
        parts.scatter_add_(1, at, p)
        if rest:
            # (masked places take the id's own value: an entry past the list may name a listed id)
            listed = torch.zeros(xs.shape[0], V + 1, dtype=torch.bool, device="cuda")
            listed.scatter_(1, torch.where(on, at, V), True)
            rho = (1 - p.sum(1)).clamp(min=0)
            parts += rho[:, None] * torch.softmax(xs.masked_fill(listed[:, :V], float("-inf")), 1)
        keep = ~none[s]
        a, b = g[s].double()[keep], g1[s].double()[keep]
        bound = 4800 * 2.0 ** -24 * (w[s, None].double() * T * parts)[keep] + 2.02 * half * torch.maximum(a.abs(), b.abs())
        assert bool(((a - b).abs() <= bound + 1e-37).all())
    rows = sorted(set(range(0, N, N // 20)) | {5, 7, N - 1})
    for i in rows:
        row = x[i].float().cpu().numpy()
        k = int(n[i])
        l, gr, dl, dg = distill_row(row, ids[i, :k].cpu().numpy(), t[i, :k].cpu().numpy(), T, rest, float(w[i]))
        for got in (loss, loss1):
            assert close(float(got[i]), l, dl), (i, float(got[i]), l, dl)
        for got in (g, g1):
            assert close(got[i].float().cpu().numpy(), gr, dg, half + 2.0 ** -23), i
