"""Operators on rows of logits, as measured cases: how a row is constrained
(penalties, biases, grammar masks), learned from (distillation from a
teacher's top logits) and made (the LM head in 8-bit integers).

Where `own` is false, `run` computes them in elementary torch operations;
where it is true, it calls the library (project-zero_b200/pz_sampling.py).

A case's "kind" names the operator:

  process   out = logits with penalties, biases and masks applied
  distill   loss of student logits against teachers' lists, with or without
            the gradient ("do": forward, train = forward then backward
            through autograd, step = loss and gradient in one call)
  head      logits = tokens (quantised per token) x 8-bit classifier rows
"""
import math
import os
import sys

import numpy as np
import torch

own = False

NEG = float("-inf")
_lib = None


def _pz():
    global _lib
    if _lib is None:
        here = os.path.dirname(os.path.abspath(__file__))
        sys.path.insert(0, os.path.join(os.path.dirname(here), "project-zero_b200"))
        import pz_sampling
        _lib = pz_sampling
    return _lib


# --------------------------------------------------------------------------
# Cases.
# --------------------------------------------------------------------------
def listed():
    return [
        # one request's decode step: a short window, a few biases, a grammar
        dict(name="process 1x128256 f32", kind="process", B=1, V=128256, dtype="f32", hist=64, ragged=False,
             bias=4, masks=1, allow=0.3, inplace=False),
        # a decode step of mixed requests: ragged windows, some rows biased,
        # some under a grammar
        dict(name="process 64x151936 bf16", kind="process", B=64, V=151936, dtype="bf16", hist=2048, ragged=True,
             bias=16, masks=5, allow=0.05, inplace=False),
        # the sampler's headline batch, every row penalised and constrained
        dict(name="process 1024x128256 f32", kind="process", B=1024, V=128256, dtype="f32", hist=1024, ragged=False,
             bias=32, masks=16, allow=0.6, inplace=False),
        # a large batch under grammars alone, in the logits buffer itself
        dict(name="mask 4096x151936 bf16 in place", kind="process", B=4096, V=151936, dtype="bf16", hist=0,
             ragged=False, bias=0, masks=32, allow=0.5, inplace=True),
        # a small micro-batch of a small vocabulary through autograd
        dict(name="distill train 16x32000 f32", kind="distill", N=16, V=32000, K=20, dtype="f32", mode="list",
             T=2.0, do="train"),
        # evaluation of a student against served log-probabilities
        dict(name="distill forward 1024x128256 f32", kind="distill", N=1024, V=128256, K=50, dtype="f32",
             mode="rest", T=1.0, do="forward"),
        # a training step through autograd, the teacher's 20 log-probabilities
        # (the most an API returns)
        dict(name="distill train 2048x151936 bf16", kind="distill", N=2048, V=151936, K=20, dtype="bf16",
             mode="rest", T=1.0, do="train"),
        # a training step that takes loss and gradient in one call
        dict(name="distill step 4096x128256 bf16", kind="distill", N=4096, V=128256, K=64, dtype="bf16",
             mode="list", T=2.0, do="step"),
        # decode of one token, the classifier of a 2B model
        dict(name="head 1x2560x128256", kind="head", B=1, dim=2560, V=128256, hidden="f32", out="f32"),
        # a decode batch
        dict(name="head 64x4096x151936", kind="head", B=64, dim=4096, V=151936, hidden="bf16", out="f32"),
        # odd sizes: a short prompt scored by a small model
        dict(name="head 301x1000x32003", kind="head", B=301, dim=1000, V=32003, hidden="f32", out="bf16"),
        # a teacher's pass over whole sequences
        dict(name="head 4096x4096x128256", kind="head", B=4096, dim=4096, V=128256, hidden="bf16", out="bf16"),
    ]


def _span(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["process", "distill", "head"])
    if kind == "process":
        V = _span(rng, 2000, 262144)
        inplace = rng.random() < 0.25
        return dict(kind=kind, B=_span(rng, 1, min(4096, 130_000_000 // V)), V=V, dtype=rng.choice(["f32", "bf16"]),
                    hist=0 if inplace else rng.choice([0, _span(rng, 1, 4096)]), ragged=rng.random() < 0.5,
                    bias=0 if inplace else rng.choice([0, _span(rng, 1, 300)]),
                    masks=rng.randint(1, 24) if inplace else rng.choice([0, rng.randint(1, 24)]),
                    allow=rng.choice([0.001, 0.1, 0.5, 0.95]), inplace=inplace)
    if kind == "distill":
        V = _span(rng, 2000, 262144)
        return dict(kind=kind, N=_span(rng, 1, min(4096, 300_000_000 // V)), V=V, K=_span(rng, 1, 256),
                    dtype=rng.choice(["f32", "bf16"]), mode=rng.choice(["list", "rest"]),
                    T=rng.choice([1.0, 2.0, rng.uniform(0.5, 4.0)]), do=rng.choice(["forward", "train", "step"]))
    V = _span(rng, 1000, 262144)
    dim = _span(rng, 256, 8192)
    return dict(kind=kind, B=_span(rng, 1, max(1, min(2048, 400_000_000_000 // (V * dim)))), dim=dim, V=V,
                hidden=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]))


# --------------------------------------------------------------------------
# Inputs.
# --------------------------------------------------------------------------
_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _logits(g, B, V, dtype):
    """Rows ~ N(0, 2.5^2) with 8 boosted ids each."""
    x = torch.randn(B, V, generator=g, device="cuda", dtype=torch.float32).mul_(2.5)
    ids = torch.randint(0, V, (B, 8), generator=g, device="cuda")
    x.scatter_add_(1, ids, torch.rand(B, 8, generator=g, device="cuda") * 10 + 5)
    return x.to(_TYPE[dtype])


def _ragged(g, B, most, ragged):
    n = torch.full((B,), most, device="cuda", dtype=torch.int64)
    if ragged:
        n = torch.randint(0, most + 1, (B,), generator=g, device="cuda")
    off = torch.zeros(B + 1, device="cuda", dtype=torch.int32)
    off[1:] = torch.cumsum(n, 0).to(torch.int32)
    return off, int(off[-1].item())


def _configs(g, B):
    """B sampler configs (temperature, top_k, top_p, repetition, frequency,
    presence, flags, reserved), penalties drawn per row."""
    c = torch.zeros(B, 8, device="cuda", dtype=torch.float32)
    c[:, 0], c[:, 2] = 0.7, 0.9
    c[:, 3] = 1.0 + 0.3 * torch.rand(B, generator=g, device="cuda")
    c[:, 4] = 0.4 * torch.rand(B, generator=g, device="cuda")
    c[:, 5] = 0.2 * torch.rand(B, generator=g, device="cuda")
    return c


def _prepare_process(c, g):
    B, V = c["B"], c["V"]
    s = dict(case=c, logits=_logits(g, B, V, c["dtype"]), cfg=None, hist=None, hist_off=None, bias_ids=None,
             bias_vals=None, bias_off=None, mask=None, mask_index=None)
    if c["hist"]:
        s["cfg"] = _configs(g, B)
        s["hist_off"], n = _ragged(g, B, c["hist"], c["ragged"])
        # a text repeats itself: half of the ids come from a few hundred
        h = torch.randint(0, V, (max(n, 1),), generator=g, device="cuda")
        few = torch.rand(max(n, 1), generator=g, device="cuda") < 0.5
        s["hist"] = torch.where(few, h % min(V, 300), h).to(torch.int32)
    if c["bias"]:
        s["bias_off"], n = _ragged(g, B, c["bias"], c["ragged"])
        s["bias_ids"] = torch.randint(0, V, (max(n, 1),), generator=g, device="cuda").to(torch.int32)
        s["bias_vals"] = torch.rand(max(n, 1), generator=g, device="cuda") * 20 - 10
    if c["masks"]:
        # half of the grammar's states allow a share of the vocabulary, the
        # others nearly all (inside a string) or nearly nothing (syntax)
        R, W = c["masks"], (V + 31) // 32
        share = torch.full((R, 1, 1), c["allow"], device="cuda")
        share[1::4], share[3::4] = 0.98, 0.0005
        bits = torch.rand(R, W, 32, generator=g, device="cuda") < share
        word = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)
        s["mask_index"] = torch.randint(0, R, (B,), generator=g, device="cuda").to(torch.int32)
        if c["ragged"]:  # rows of requests without a grammar
            s["mask_index"][torch.rand(B, generator=g, device="cuda") < 0.3] = -1
    s["n_allowed"] = torch.empty(B, device="cuda", dtype=torch.int32)
    s["out"] = s["logits"] if c["inplace"] else torch.empty_like(s["logits"])
    return s


def _prepare_distill(c, g):
    N, V, K = c["N"], c["V"], min(c["K"], c["V"])
    x = torch.randn(N, V, generator=g, device="cuda", dtype=torch.float32).mul_(2.5)
    # the teacher's ids, distinct in a row, and where the student is high too
    first = torch.randint(0, V, (N, 1), generator=g, device="cuda")
    step = torch.randint(1, max(2, V // K), (N, 1), generator=g, device="cuda")
    j = torch.arange(K, device="cuda")
    ids = (first + step * j) % V
    x.scatter_add_(1, ids, torch.rand(N, K, generator=g, device="cuda") * (12.0 * torch.exp(-j / 12.0) + 2))
    t = (torch.randn(N, K, generator=g, device="cuda") * 2.0 + 9.0 * torch.exp(-j / 8.0)).sort(1, descending=True)[0]
    if c["mode"] == "rest":
        # log-probabilities over the whole vocabulary: 2 to 30 % are off the list
        rest = 0.02 + 0.28 * torch.rand(N, 1, generator=g, device="cuda")
        t = torch.log_softmax(t, 1) + torch.log1p(-rest)
    n = torch.where(torch.rand(N, generator=g, device="cuda") < 0.8, K,
                    torch.randint(1, K + 1, (N,), generator=g, device="cuda"))
    past = j[None, :] >= n[:, None]
    w = torch.full((N,), 1.0 / N, device="cuda")
    if N > 1:  # prompt positions and padding carry no weight
        w[torch.rand(N, generator=g, device="cuda") < 0.1] = 0.0
    s = dict(case=c, logits=x.to(_TYPE[c["dtype"]]), ids=ids.masked_fill(past, -1).to(torch.int32).contiguous(),
             values=t.masked_fill(past, NEG).contiguous(), weight=w,
             loss=torch.empty(N, device="cuda"))
    if c["do"] == "train":
        s["logits"].requires_grad_(True)
        s["up"] = 0.5 + torch.rand(N, generator=g, device="cuda")
    if c["do"] == "step":
        s["grad"] = torch.empty_like(s["logits"])
    return s


def _padded(rows, cols):
    """An int8 [rows, cols] view of rows that are 16 bytes apart or a
    multiple of it."""
    return torch.zeros(rows, (cols + 15) // 16 * 16, device="cuda", dtype=torch.int8)[:, :cols]


def _prepare_head(c, g):
    B, dim, V = c["B"], c["dim"], c["V"]
    hidden = torch.randn(B, dim, generator=g, device="cuda") * (0.5 + torch.rand(1, dim, generator=g, device="cuda"))
    w_q, w_scale = _padded(V, dim), torch.empty(V, device="cuda")
    w = torch.randn(V, dim, generator=g, device="cuda").mul_(0.02)
    top = w.abs().amax(1)
    w_scale.copy_(top / 127)
    w_q.copy_(w.mul_((127 / top)[:, None]).round_())
    return dict(case=c, hidden=hidden.to(_TYPE[c["hidden"]]), w_q=w_q, w_scale=w_scale,
                hidden_q=_padded(B, dim), hidden_scale=torch.empty(B, device="cuda"),
                logits=torch.empty(B, V, device="cuda", dtype=_TYPE[c["out"]]))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"process": _prepare_process, "distill": _prepare_distill, "head": _prepare_head}[case["kind"]](case, g)


# --------------------------------------------------------------------------
# Plain forms.
# --------------------------------------------------------------------------
def _row_of(off, n):
    """The row of each of the n entries of a list with these offsets."""
    return torch.repeat_interleave(torch.arange(off.numel() - 1, device=off.device), off.diff().long(), output_size=n)


def _plain_process(s):
    logits = s["logits"]
    B, V = logits.shape
    x = logits.float()
    if s["hist"] is not None and s["hist_off"] is not None:
        n = s["hist"].numel() if s["case"]["ragged"] is False else int(s["hist_off"][-1])
        row, t = _row_of(s["hist_off"], n), s["hist"][:n].long()
        fine = (t >= 0) & (t < V)
        count = torch.zeros(B * V, device=x.device)
        count.scatter_add_(0, torch.where(fine, row * V + t, 0), fine.float())
        count = count.view(B, V)
        rep, freq, pres = (s["cfg"][:, k:k + 1] for k in (3, 4, 5))
        y = torch.where(rep == 1, x, torch.where(x > 0, x / rep, x * rep))
        x = torch.where(count > 0, y - (count * freq + pres), x)
    if s["bias_ids"] is not None:
        n = s["bias_ids"].numel() if s["case"]["ragged"] is False else int(s["bias_off"][-1])
        row, t = _row_of(s["bias_off"], n), s["bias_ids"][:n].long()
        last = torch.full((B * V,), -1, device=x.device, dtype=torch.int32)
        last.scatter_reduce_(0, row * V + t, torch.arange(n, device=x.device, dtype=torch.int32), "amax")
        last = last.view(B, V)
        x = torch.where(last >= 0, x + s["bias_vals"][last.clamp(min=0)], x)
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        bits = bits.view(s["mask"].shape[0], -1)[:, :V].bool()
        at = s["mask_index"].long()
        allowed = bits[at.clamp(min=0)] | (at < 0)[:, None]
        x = torch.where(allowed, x, NEG)
        s["n_allowed"].copy_(allowed.sum(1))
    else:
        s["n_allowed"].fill_(V)
    s["out"].copy_(x)
    return s["out"], s["n_allowed"]


def _plain_distill(s):
    c, T = s["case"], s["case"]["T"]
    ids, values, w = s["ids"], s["values"], s["weight"]
    x = s["logits"].detach().float() / T
    N, V = x.shape
    fine = (ids >= 0) & (ids < V)
    at = torch.where(fine, ids, 0).long()
    off_list = torch.ones_like(x, dtype=torch.bool)
    off_list.scatter_(1, at, ~fine)  # an ignored entry leaves id 0 as it is unless the row lists it
    off_list[:, 0] = ~((ids == 0) & fine).any(1)
    if c["mode"] == "list":
        t = values.masked_fill(~fine, NEG) / T
        p = torch.exp(t - t.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        rho = torch.zeros(N, device=x.device)
    else:
        p = torch.exp(values).masked_fill(~fine, 0)
        rho = (1 - p.sum(1)).clamp(min=0)
    e = torch.exp(x - x.amax(1, keepdim=True))
    total = e.sum(1)
    rest = torch.where(off_list, e, 0).sum(1)
    log_q = x.gather(1, at) - x.amax(1, keepdim=True) - total.log()[:, None]
    loss = torch.where(p > 0, p * (p.log() - log_q), 0).sum(1)
    loss = loss + torch.where(rho > 0, rho * (rho.log() - rest.log() + total.log()), 0)
    s["loss"].copy_(torch.where(w != 0, w * (T * T) * loss, 0))
    if c["do"] == "forward":
        return (s["loss"],)
    mass = (p.sum(1) + rho if c["mode"] == "rest" else torch.ones_like(rho))[:, None]
    grad = e * (mass / total[:, None] - torch.where(off_list, (rho / rest)[:, None], 0))
    grad = grad.scatter_add_(1, at, -p)
    by = w * T * s["up"] if c["do"] == "train" else w * T
    grad = torch.where(w[:, None] != 0, grad * by[:, None], 0)
    if c["do"] == "step":
        s["grad"].copy_(grad)
        return s["loss"], s["grad"]
    return s["loss"], grad.to(s["logits"].dtype)


def _plain_head(s):
    x = s["hidden"].float()
    B, dim = x.shape
    top = x.abs().amax(1)
    most = torch.full_like(top, 127)  # (a division by a Python number would be a product with its reciprocal)
    scale = top / most
    q = (x * (most / top)[:, None]).round()
    # sums of 1024 products of 8-bit values are whole numbers below 2^24:
    # exact in 32-bit floats; the sums of those are taken in whole numbers
    pieces = -(-dim // 1024)
    pad = (0, pieces * 1024 - dim)
    a = torch.nn.functional.pad(q, pad).view(B, pieces, 1024).transpose(0, 1)
    b = torch.nn.functional.pad(s["w_q"].float(), pad).view(-1, pieces, 1024).permute(1, 2, 0)
    total = torch.bmm(a, b).to(torch.int32).sum(0, dtype=torch.int32)
    s["logits"].copy_(total.float() * (scale[:, None] * s["w_scale"][None, :]))
    return (s["logits"],)


# --------------------------------------------------------------------------
# The library's calls.
# --------------------------------------------------------------------------
def _own_process(s):
    _pz().process_logits(s["logits"], s["out"], cfg=s["cfg"], hist=s["hist"], hist_off=s["hist_off"],
                         bias_ids=s["bias_ids"], bias_vals=s["bias_vals"], bias_off=s["bias_off"], mask=s["mask"],
                         mask_index=s["mask_index"], n_allowed=s["n_allowed"])
    return s["out"], s["n_allowed"]


def _own_distill(s):
    pz, c = _pz(), s["case"]
    how = dict(weight=s["weight"], temperature=c["T"], mode=pz.DISTILL_LIST if c["mode"] == "list" else pz.DISTILL_REST)
    if c["do"] == "forward":
        pz.distill_forward(s["logits"], s["ids"], s["values"], s["loss"], **how)
        return (s["loss"],)
    if c["do"] == "step":
        pz.distill_loss_grad(s["logits"], s["ids"], s["values"], s["loss"], s["grad"], **how)
        return s["loss"], s["grad"]
    loss = pz.distill_loss(s["logits"], s["ids"], s["values"], **how)
    grad, = torch.autograd.grad(loss, s["logits"], s["up"])
    return loss, grad


def _own_head(s):
    _pz().lm_head_i8(s["hidden"], s["w_q"], s["w_scale"], s["logits"], s["hidden_q"], s["hidden_scale"])
    return (s["logits"],)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"process": _own_process, "distill": _own_distill, "head": _own_head}[kind](state)
    return {"process": _plain_process, "distill": _plain_distill, "head": _plain_head}[kind](state)


# --------------------------------------------------------------------------
# What a pass cannot do without.
# --------------------------------------------------------------------------
_SIZE = {"f32": 4, "bf16": 2}


def work(case):
    c = case
    if c["kind"] == "process":
        B, V, es = c["B"], c["V"], _SIZE[c["dtype"]]
        part = 0.5 if c["ragged"] else 1.0
        small = B * part * (4 * c["hist"] + 8 * c["bias"]) + (40 * B if c["hist"] else 0) + 4 * B
        if c["masks"]:
            small += c["masks"] * ((V + 31) // 32) * 4 + 4 * B
        if c["inplace"]:  # only the ids that a mask takes are written
            shares = [c["allow"], 0.98, c["allow"], 0.0005]
            mean = sum(shares[k % 4] for k in range(c["masks"])) / c["masks"]
            return {"bytes": small + B * V * es * (1 - mean), "flops": 0}
        return {"bytes": small + 2 * B * V * es, "flops": 4 * B * part * (c["hist"] + c["bias"])}
    if c["kind"] == "distill":
        N, V, K, es = c["N"], c["V"], c["K"], _SIZE[c["dtype"]]
        passes = {"forward": 1, "step": 2, "train": 3}[c["do"]]
        return {"bytes": N * V * es * passes + N * (8 * K + 8), "flops": N * V * (3 if c["do"] == "forward" else 7)}
    B, dim, V = c["B"], c["dim"], c["V"]
    return {"bytes": V * (dim + 4) + B * dim * _SIZE[c["hidden"]] + B * V * _SIZE[c["out"]], "flops": 2 * B * dim * V}


# --------------------------------------------------------------------------
# The operators' definitions in 64 bits.
# --------------------------------------------------------------------------
def _exact_process(s):
    x = s["logits"].double()
    B, V = x.shape
    flat = x.view(-1)
    if s["hist"] is not None:
        off = s["hist_off"].long()
        n = int(off[-1])
        row = torch.searchsorted(off, torch.arange(n, device=x.device), right=True) - 1
        at, count = torch.unique(row * V + s["hist"][:n].long(), return_counts=True)
        cfg = s["cfg"].double()[at // V]
        v, rep = flat[at], cfg[:, 3]
        v = torch.where(v > 0, v / rep, v * rep) - (count * cfg[:, 4] + cfg[:, 5])
        flat[at] = v
    if s["bias_ids"] is not None:
        off, ids, vals = (s[k].cpu().numpy() for k in ("bias_off", "bias_ids", "bias_vals"))
        for r in range(B):
            last = {int(t): float(b) for t, b in zip(ids[off[r]:off[r + 1]], vals[off[r]:off[r + 1]])}
            if last:
                x[r, torch.tensor(list(last), device=x.device)] += torch.tensor(list(last.values()), device=x.device,
                                                                                  dtype=torch.float64)
    left = torch.full((B,), V, device=x.device, dtype=torch.int32)
    if s["mask"] is not None:
        raw = s["mask"].cpu().numpy().view(np.uint8)
        bits = torch.from_numpy(np.unpackbits(raw, axis=1, bitorder="little")[:, :V].copy()).to(x.device).bool()
        for k in range(bits.shape[0]):
            rows = (s["mask_index"] == k).nonzero()[:, 0]
            if rows.numel():
                x[rows] = x[rows].masked_fill(~bits[k], NEG)
                left[rows] = int(bits[k].sum())
    return x, left


def _exact_distill(s):
    c, T = s["case"], s["case"]["T"]
    N, V = s["logits"].shape
    every = []
    for r in range(0, N, 256):
        x = s["logits"].detach()[r:r + 256].double() / T
        ids, t, w = s["ids"][r:r + 256].long(), s["values"][r:r + 256].double(), s["weight"][r:r + 256].double()
        fine = ids >= 0
        if c["mode"] == "list":
            p = torch.softmax((t / T).masked_fill(~fine, NEG), 1)
            rho = None
        else:
            p = t.exp().masked_fill(~fine, 0)
            rho = (1 - p.sum(1)).clamp(min=0)
        # the target as a row over V and one more place for ignored entries
        wide = torch.zeros(x.shape[0], V + 1, device=x.device, dtype=torch.float64)
        at = torch.where(fine, ids, V)
        target = wide.scatter_add(1, at, p)[:, :V]
        on = wide.scatter(1, at, 1.0)[:, :V] > 0
        log_q = torch.log_softmax(x, 1)
        loss = (torch.special.xlogy(target, target) - target * log_q).sum(1)
        grad = log_q.exp()
        if rho is not None:
            among = torch.log_softmax(x.masked_fill(on, NEG), 1)
            r_log = torch.logsumexp(log_q.masked_fill(on, NEG), 1)
            loss = loss + torch.where(rho > 0, rho * (rho.log() - r_log), 0)
            grad = grad * (p.sum(1) + rho)[:, None]
            target = target + rho[:, None] * among.exp()
        by = w * T * (s["up"][r:r + 256].double() if c["do"] == "train" else 1)
        loss = w * T * T * loss
        every.append((loss, None if c["do"] == "forward" else (grad - target) * by[:, None]))
    loss = torch.cat([a for a, _ in every])
    return (loss,) if c["do"] == "forward" else (loss, torch.cat([b for _, b in every]))


def _exact_head(s):
    # the quantisation is defined by its 32-bit steps: each is taken in 64
    # bits and rounded to 32 once
    x = s["hidden"].double()
    top = x.abs().amax(1, keepdim=True)
    scale, inv = (top / 127).float().double(), (127 / top).float().double()
    q = torch.round((x * inv).float().double())
    return ((q @ s["w_q"].double().T) * scale * s["w_scale"].double()[None, :],)


def exact(case, seed):
    s = prepare(case, seed)
    return {"process": _exact_process, "distill": _exact_distill, "head": _exact_head}[case["kind"]](s)
