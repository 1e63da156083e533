"""Cases of the draft-verification operators: greedy and sampled verification
from the target's logits, verification from probabilities, and the target's
probabilities themselves.

``run`` computes them in elementary torch operations, or, with ``own`` set,
makes the calls a user makes of ``suffixgpu_b200.ops``. ``exact`` restates
the definitions in 64 bits in another way.

Definitions (one logits row l, NaN read as -inf, m its largest value):
w_i = exp((l_i - m) / T); top_k keeps the values >= the k-th largest; top_p
keeps, of those, the values >= t, t the largest value whose tokens >= t hold
at least p of the kept mass; P = w over the kept mass. T <= 0: all mass on
the first largest token. Draft j is accepted while u_j * q_j(x_j) < P_j(x_j)
(q = 1 without draft probabilities); the row s of the first rejection (or
the row after the last draft) gives one more token, drawn by u_K from P_s
without the rejected token (from max(P_s - q_s, 0) with draft
probabilities).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16,
          "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one stream drafting 4 tokens, deterministic decoding: latency
        dict(name="greedy_b1", op="greedy", b=1, k=4, v=32000, dtype="bf16",
             ragged=False, accept=0.7),
        # an odd vocabulary, 32-bit logits, only the drafted rows stored
        dict(name="greedy_odd_ragged", op="greedy", b=37, k=7, v=50021,
             dtype="fp32", ragged=True, accept=0.6),
        # the 256-row decode batch with 16 drafts a row
        dict(name="greedy_b256", op="greedy", b=256, k=16, v=128256,
             dtype="bf16", ragged=False, accept=0.75),
        # plain decoding of one stream: no drafts, one token to sample
        dict(name="sampled_b1_single", op="sampled", b=1, k=0, v=128256,
             dtype="bf16", ragged=False, accept=0.7, temps="one",
             filters="none"),
        # the 256-row decode batch, greedy and sampled requests mixed
        dict(name="sampled_b256", op="sampled", b=256, k=16, v=128256,
             dtype="bf16", ragged=False, accept=0.75, temps="mixed",
             filters="none"),
        # top-p for every request, as servers default to; odd vocabulary
        dict(name="sampled_topp_odd", op="sampled", b=24, k=5, v=50021,
             dtype="fp16", ragged=True, accept=0.7, temps="mixed",
             filters="p"),
        # the drafter with 32 drafts, every request with its own top-k, top-p
        dict(name="sampled_topkp_b128", op="sampled", b=128, k=32, v=128256,
             dtype="bf16", ragged=False, accept=0.8, temps="mixed",
             filters="kp"),
        # probabilities in hand, drafts without a distribution: latency
        dict(name="probs_onehot_b8", op="probs", b=8, k=16, v=32000,
             dtype="fp32", ragged=False, accept=0.7, qprobs=False),
        # a drafter with a distribution of its own over the vocabulary
        dict(name="probs_q_b64", op="probs", b=64, k=16, v=128256,
             dtype="fp32", ragged=False, accept=0.7, qprobs=True),
        # the next token's distribution of one stream
        dict(name="target_b1", op="target", b=1, k=0, v=32000, dtype="fp32",
             ragged=False, accept=0.7, temps="one", filters="none"),
        # the distributions of 64 requests with 16 drafts each
        dict(name="target_b64", op="target", b=64, k=16, v=128256,
             dtype="bf16", ragged=False, accept=0.7, temps="mixed",
             filters="none"),
        # the same with both filters, 32-bit logits of an odd vocabulary
        dict(name="target_topkp_odd", op="target", b=32, k=5, v=100003,
             dtype="fp32", ragged=False, accept=0.7, temps="mixed",
             filters="kp"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["greedy", "sampled", "probs", "target"])
    b = _log_int(rng, 1, 256)
    k = rng.randint(0, 32)
    v = min(131072, _log_int(rng, 500, 131072) | rng.randint(0, 1))
    most = 100_000_000 if op in ("probs", "target") else 400_000_000
    while b * (k + 1) * v > most:
        if k > 4:
            k //= 2
        else:
            b = max(1, b // 2)
    case = dict(op=op, b=b, k=k, v=v, dtype=rng.choice(sorted(DTYPES)),
                ragged=rng.random() < 0.5,
                accept=round(rng.uniform(0.3, 0.95), 3))
    if op in ("sampled", "target"):
        case["temps"] = rng.choice(["one", "mixed"])
        case["filters"] = rng.choice(["none", "p", "k", "kp"])
    if op == "probs":
        case["dtype"] = "fp32"
        case["qprobs"] = rng.random() < 0.5
    if op == "target":
        case["ragged"] = False
    return case


def _expected_rows(case):
    """Expected logits rows a request needs: the accepted drafts' and one."""
    k = case["k"]
    if case["op"] == "target":
        return k + 1.0
    a = case["accept"]
    if case["op"] != "greedy":  # a token of probability p is accepted with p
        a = 0.85 * a + 0.15 * (1 - a)

    def rows(n):
        return sum(a ** j for j in range(n + 1))
    return 0.7 * rows(k) + 0.3 * sum(rows(n) for n in range(k + 1)) / (k + 1)


def work(case):
    b, k, v = case["b"], case["k"], case["v"]
    rows = b * _expected_rows(case)
    size = SIZE[case["dtype"]]
    small = 4 * b * (3 * k + 4)
    if case["op"] == "greedy":  # one comparison a logit
        return {"bytes": rows * v * size + small, "flops": rows * v}
    if case["op"] == "sampled":  # difference, scale, exp, sum
        return {"bytes": rows * v * size + small, "flops": 4 * rows * v}
    if case["op"] == "target":  # and the scale and the store of each
        return {"bytes": rows * v * (size + 4) + small, "flops": 5 * rows * v}
    # one row a request (its residual summed), a gather a draft
    rows_b = 2 if case["qprobs"] else 1
    return {"bytes": b * v * 4 * rows_b + small, "flops": 2 * b * v}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _logits_rows(g, n, v, drafted, p_draft, masked, dtype):
    """n rows of logits: a broad bulk, a few likely tokens, the drafted token
    (-1: none) at probability p_draft, and, for masked rows, a grammar's mask
    that leaves about a tenth of the vocabulary."""
    out = torch.empty(n, v, dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // v)
    for lo in range(0, n, step):
        hi = min(n, lo + step)
        m = hi - lo
        x = torch.randn(m, v, generator=g, device="cuda") * 2.5
        drop = (_rand(g, m, v) < 0.9) & masked[lo:hi, None]
        x.masked_fill_(drop, -math.inf)
        top = math.log(v) + 3.1
        fav = torch.randint(0, v, (m, 6), generator=g, device="cuda")
        x.scatter_(1, fav, top - 4.0 * _rand(g, m, 6))
        z = torch.logsumexp(x, dim=1, keepdim=True)
        d = drafted[lo:hi].long()
        p = p_draft[lo:hi, None]
        val = z + torch.log(p / (1 - p))
        have = (d >= 0)[:, None]
        idx = d.clamp(min=0)[:, None]
        x.scatter_(1, idx, torch.where(have, val, x.gather(1, idx)))
        out[lo:hi] = x.to(dtype)
    return out


def prepare(case, seed):
    b, k, v = case["b"], case["k"], case["v"]
    g = _gen(seed)
    nv = torch.where(_rand(g, b) < 0.7, torch.full((b,), k, device="cuda"),
                     torch.randint(0, k + 1, (b,), generator=g,
                                   device="cuda")).to(torch.int32)
    draft = torch.randint(0, v, (b, k), generator=g, device="cuda",
                          dtype=torch.int32)
    j = torch.arange(k, device="cuda")
    draft = torch.where(j[None, :] < nv[:, None], draft,
                        torch.full_like(draft, -1))
    likely = _rand(g, b, k + 1) < case["accept"]
    p = torch.where(likely, 0.7 + 0.29 * _rand(g, b, k + 1),
                    0.001 + 0.299 * _rand(g, b, k + 1))
    masked = (_rand(g, b) < 0.125)[:, None].expand(b, k + 1)
    drafted = torch.cat([draft, draft.new_full((b, 1), -1)], dim=1)
    if case["ragged"]:  # the rows 0..num_valid of each request, packed
        keep = torch.arange(k + 1, device="cuda")[None, :] <= nv[:, None]
        start = torch.cumsum(nv + 1, 0) - (nv + 1)
        start = start.to(torch.int32)
    else:
        keep = torch.ones(b, k + 1, dtype=torch.bool, device="cuda")
        start = None
    dtype = DTYPES[case["dtype"]]
    rows = _logits_rows(g, int(keep.sum()), v, drafted[keep], p[keep],
                        masked[keep], dtype)
    st = {"op": case["op"], "draft": draft, "nv": nv, "start": start,
          "u": _rand(g, b, k + 1)}
    if case["op"] == "probs":
        rows = torch.softmax(rows, dim=1)
        if case["qprobs"]:
            # a flatter distribution near the target's, and drafts from it
            q = torch.empty(b, k, v, device="cuda")
            view = None if case["ragged"] else rows.view(b, k + 1, v)
            for i in range(k):
                if view is None:
                    at = (start.long() + i).clamp(max=rows.shape[0] - 1)
                    src = rows[at]
                else:
                    src = view[:, i]
                qi = src.sqrt() * (0.5 + _rand(g, b, v))
                q[:, i] = qi / qi.sum(1, keepdim=True)
                x = torch.multinomial(q[:, i], 1, generator=g)[:, 0]
                draft[:, i] = torch.where(i < nv, x.to(torch.int32),
                                          draft[:, i])
            st["q"] = q
        else:
            st["q"] = None
    st["rows"] = rows if case["ragged"] else rows.view(b, k + 1, v)
    if case["op"] in ("sampled", "target"):
        if case["temps"] == "one":
            st["temperature"] = 1.0
        else:
            t = 0.5 + 0.8 * _rand(g, b)
            st["temperature"] = torch.where(_rand(g, b) < 0.125,
                                            torch.zeros_like(t), t)
        f = case["filters"]
        st["top_p"] = st["top_k"] = None
        if "p" in f and f != "none":
            st["top_p"] = 0.7 + 0.3 * _rand(g, b)
        if "k" in f:
            st["top_k"] = torch.randint(1, 200, (b,), generator=g,
                                        device="cuda", dtype=torch.int32)
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _per_request(x, b, dtype, default):
    if x is None:
        x = default
    if not torch.is_tensor(x):
        return torch.full((b,), x, dtype=dtype, device="cuda")
    return x.to(dtype)


def _plain_rows(st, j):
    """Row j of every request [B, V] (a request without one gets another
    request's, which nothing then uses)."""
    if st["start"] is None:
        return st["rows"][:, j]
    at = (st["start"].long() + j).clamp(max=st["rows"].shape[0] - 1)
    return st["rows"][at]


def _plain_probs(x, temperature, top_k, top_p):
    """[B, V] probabilities in 64 bits: sums next to a border decide."""
    b, v = x.shape
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    m = x.max(dim=1, keepdim=True).values
    t = temperature[:, None].double()
    w = torch.exp((x - m) / torch.where(t > 0, t, 1.0))
    w = torch.where(x == m, 1.0, w)
    w = torch.where(x == -math.inf, 0.0, w)
    if top_k is not None or top_p is not None:
        sx, order = torch.sort(x, dim=1, descending=True)
        low = torch.full((b, 1), -math.inf, dtype=torch.float64,
                         device="cuda")
        if top_k is not None:
            kk = top_k.long()[:, None]
            kth = sx.gather(1, (kk.clamp(1, v) - 1))
            low = torch.where((kk > 0) & (kk < v), kth, low)
        sw = w.gather(1, order)
        sw = torch.where(sx >= low, sw, 0.0)
        if top_p is not None:
            pp = top_p.double()[:, None]
            cum = torch.cumsum(sw, dim=1)
            need = pp * sw.sum(dim=1, keepdim=True)
            first = (cum < need).sum(dim=1, keepdim=True).clamp(max=v - 1)
            tp = torch.where(pp > 0, sx.gather(1, first), m)
            low = torch.where(pp < 1, torch.maximum(low, tp), low)
        w = torch.where(x >= low, w, 0.0)
    z = w.sum(dim=1, keepdim=True)
    p = w / torch.where(z > 0, z, 1.0)
    one = torch.zeros_like(p)
    one.scatter_(1, x.argmax(dim=1, keepdim=True), 1.0)
    return torch.where(t > 0, p, torch.where(m > -math.inf, one, 0.0))


def _plain_softmax(x, temperature):
    """[N, V] probabilities without filters, in 32 bits."""
    x = x.float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    m = x.max(dim=1, keepdim=True).values
    t = temperature[:, None]
    w = torch.exp((x - m) / torch.where(t > 0, t, 1.0))
    w = torch.where(x == m, 1.0, w)
    w = torch.where(x == -math.inf, 0.0, w)
    z = w.sum(dim=1, keepdim=True)
    p = w / torch.where(z > 0, z, 1.0)
    one = torch.zeros_like(p)
    one.scatter_(1, x.argmax(dim=1, keepdim=True), 1.0)
    return torch.where(t > 0, p, torch.where(m > -math.inf, one, 0.0))


def _plain_draw(r, u):
    """First index whose running sum of r [B, V] passes u * its total; -1
    for a row without mass."""
    cum = torch.cumsum(r, dim=1)
    total = cum[:, -1:]
    i = (cum <= u.double()[:, None] * total).sum(dim=1)
    v = r.shape[1]
    last = v - 1 - (r.flip(1) > 0).to(torch.int8).argmax(dim=1)
    i = torch.minimum(i, last)
    return torch.where(total[:, 0] > 0, i, -1).to(torch.int32)


def _plain_emit(st, probs_of, draw_of):
    """The acceptance chain over positions: probs_of(j) -> [B, V], draw_of(
    p, j, x, rejected) -> the token that follows."""
    draft, nv, u = st["draft"], st["nv"], st["u"]
    b, k = draft.shape
    out = torch.full((b, k + 1), -1, dtype=torch.int32, device="cuda")
    alive = nv >= 0
    count = torch.zeros(b, dtype=torch.int32, device="cuda")
    for j in range(k + 1):
        p = probs_of(j)
        if j < k:
            x = draft[:, j].long()
            inside = (x >= 0) & (x < p.shape[1])
            xi = x.clamp(0, p.shape[1] - 1)[:, None]
            px = p.gather(1, xi)[:, 0]
            qx = 1.0
            if st.get("q") is not None:
                qx = st["q"][:, j].gather(1, xi)[:, 0].double()
            drafted = j < nv
            ok = inside & drafted & (u[:, j].double() * qx < px)
        else:
            x = torch.full((b,), -1, device="cuda")
            drafted = torch.zeros(b, dtype=torch.bool, device="cuda")
            ok = drafted
        tok = draw_of(p, j, x, drafted)
        val = torch.where(ok, x.to(torch.int32), tok)
        out[:, j] = torch.where(alive, val, out[:, j])
        count += (alive & (val >= 0)).to(torch.int32)
        alive = alive & ok
    return out, count


def _without(p, x, drafted):
    """P without the rejected draft; all of P if nothing else is left."""
    v = p.shape[1]
    hit = drafted & (x >= 0) & (x < v)
    r = p.scatter(1, x.clamp(0, v - 1)[:, None], 0.0)
    r = torch.where(hit[:, None], r, p)
    return torch.where(r.sum(1, keepdim=True) > 0, r, p)


def _plain(st):
    op = st["op"]
    if op == "target":
        b, j, v = st["rows"].shape
        t = _per_request(st["temperature"], b, torch.float32, 1.0)
        out = torch.empty(b, j, v, device="cuda")
        for i in range(j):
            if st["top_k"] is None and st["top_p"] is None:
                out[:, i] = _plain_softmax(st["rows"][:, i], t)
            else:
                out[:, i] = _plain_probs(st["rows"][:, i], t, st["top_k"],
                                         st["top_p"]).float()
        return {"probs": out}
    if op == "greedy":
        def one_hot(j):
            x = _plain_rows(st, j).float()
            x = torch.where(torch.isnan(x), -math.inf, x)
            p = torch.zeros_like(x)
            p.scatter_(1, x.argmax(dim=1, keepdim=True), 1.0)
            return torch.where(x.max(1, keepdim=True).values > -math.inf, p,
                               0.0)

        def first(p, j, x, drafted):
            return torch.where(p.sum(1) > 0, p.argmax(dim=1),
                               -1).to(torch.int32)
        out, count = _plain_emit(dict(st, u=torch.zeros_like(st["u"])),
                                 one_hot, first)
        return {"sampled": out, "count": count}
    if op == "sampled":
        t = _per_request(st["temperature"], st["draft"].shape[0],
                         torch.float32, 1.0)
        out, count = _plain_emit(
            st, lambda j: _plain_probs(_plain_rows(st, j), t, st["top_k"],
                                       st["top_p"]),
            lambda p, j, x, drafted: _plain_draw(_without(p, x, drafted),
                                                 st["u"][:, -1]))
        return {"sampled": out, "count": count}

    def draw_of(p, j, x, drafted):
        if st["q"] is None or j == st["draft"].shape[1]:
            r = _without(p, x, drafted)
        else:
            r = (p - st["q"][:, j].double()).clamp(min=0.0)
            r = torch.where(drafted[:, None] & (r.sum(1, keepdim=True) > 0),
                            r, p)
        return _plain_draw(r, st["u"][:, -1])
    out, count = _plain_emit(
        st, lambda j: _plain_rows(st, j).double(), draw_of)
    return {"sampled": out, "count": count}


def run(state):
    if not own:
        return _plain(state)
    from suffixgpu_b200 import ops
    op = state["op"]
    if op == "target":
        return {"probs": ops.target_probs(
            state["rows"], state["temperature"], top_k=state["top_k"],
            top_p=state["top_p"])}
    if op == "greedy":
        out, count = ops.verify_greedy(state["rows"], state["draft"],
                                       num_valid=state["nv"],
                                       row_start=state["start"])
    elif op == "sampled":
        out, count = ops.verify_sampled(
            state["rows"], state["draft"], state["u"],
            num_valid=state["nv"], temperature=state["temperature"],
            top_k=state["top_k"], top_p=state["top_p"],
            row_start=state["start"])
    else:
        out, count = ops.verify_probs(state["rows"], state["draft"],
                                      state["u"], num_valid=state["nv"],
                                      draft_probs=state["q"],
                                      row_start=state["start"])
    return {"sampled": out, "count": count}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, one request (or row) after another
# ---------------------------------------------------------------------------
def _exact_log_probs(x, t, k, p):
    """Log-probabilities of one row [V] in 64 bits, by the distinct values of
    the row: a table of values, their counts and their masses."""
    x = x.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    out = torch.full_like(x, -math.inf)
    if not bool((x > -math.inf).any()):
        return out
    if not t > 0:
        out[int(torch.nonzero(x == x.max())[0])] = 0.0
        return out
    vals, inv, num = torch.unique(x, return_inverse=True, return_counts=True)
    if math.isinf(float(vals[-1])):
        lw = torch.where(vals == vals[-1], 0.0, -math.inf).double()
    else:
        lw = (vals - vals[-1]) / t
    above = torch.flip(torch.cumsum(torch.flip(num, [0]), 0), [0]) - num
    keep = torch.ones_like(vals, dtype=torch.bool)
    if k is not None and 0 < k < x.numel():
        keep &= above < k
    if p is not None and p < 1:
        mass = torch.where(keep, num * torch.exp(lw), 0.0)
        over = torch.flip(torch.cumsum(torch.flip(mass, [0]), 0), [0]) - mass
        if p > 0:
            keep &= over < p * mass.sum()
        else:
            keep &= vals == vals[-1]
    lw = torch.where(keep, lw, -math.inf)
    lz = torch.logsumexp(lw + torch.log(num.double()), 0)
    return (lw - lz)[inv]


def _exact_draw(r, u):
    total = r.sum()
    if not float(total) > 0:
        return -1
    cum = torch.cumsum(r / total, 0)
    i = int(torch.searchsorted(cum, torch.tensor(float(u), device="cuda",
                                                 dtype=torch.float64),
                               right=True))
    return min(i, int(torch.nonzero(r)[-1]))


def exact(case, seed):
    st = prepare(case, seed)
    b, k, v = case["b"], case["k"], case["v"]
    f_t = st.get("temperature")
    ts = ([float(f_t)] * b if not torch.is_tensor(f_t) else
          f_t.double().tolist()) if f_t is not None else [0.0] * b
    ks = st["top_k"].tolist() if st.get("top_k") is not None else [None] * b
    ps = (st["top_p"].double().tolist() if st.get("top_p") is not None
          else [None] * b)
    if case["op"] == "target":
        out = torch.empty(b, k + 1, v, dtype=torch.float64, device="cuda")
        for i in range(b):
            for j in range(k + 1):
                out[i, j] = torch.exp(_exact_log_probs(
                    st["rows"][i, j], ts[i], ks[i], ps[i]))
        return {"probs": out}
    nv = st["nv"].tolist()
    draft = st["draft"].tolist()
    u = st["u"].double().tolist()
    start = None if st["start"] is None else st["start"].tolist()
    sampled, count = [], []
    for i in range(b):
        got = []
        for j in range(nv[i] + 1):
            row = (st["rows"][i, j] if start is None
                   else st["rows"][start[i] + j])
            if case["op"] == "probs":
                p = row.double()
            else:
                p = torch.exp(_exact_log_probs(row, ts[i], ks[i], ps[i]))
            x = draft[i][j] if j < nv[i] else -1
            q = None
            if x >= 0 and st.get("q") is not None:
                q = st["q"][i, j].double()
            if x >= 0:
                qx = 1.0 if q is None else float(q[x])
                uj = 0.0 if case["op"] == "greedy" else u[i][j]
                if uj * qx < float(p[x]):
                    got.append(x)
                    continue
                r = p.clone() if q is None else (p - q).clamp(min=0)
                if q is None:
                    r[x] = 0.0
                p = r if float(r.sum()) > 0 else p
            tok = _exact_draw(p, 0.0 if case["op"] == "greedy" else u[i][k])
            got += [tok] if tok >= 0 else []
            break
        sampled.append(got + [-1] * (k + 1 - len(got)))
        count.append(len(got))
    return {"sampled": torch.tensor(sampled, dtype=torch.int32),
            "count": torch.tensor(count, dtype=torch.int32)}
