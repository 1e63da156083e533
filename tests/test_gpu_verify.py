"""Draft verification on the GPU against the 64-bit oracle: tokens and counts
are equal, probabilities agree to fp32 rounding."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import suffix_oracle as so
from oracle import verify_oracle as vo
from suffixgpu_b200 import SuffixGPUDrafter, ops
from suffixgpu_b200 import workloads as wl

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DT = [torch.float32, torch.bfloat16, torch.float16]
NEG = float("-inf")


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy().astype(np.float64)


def _case(seed, b, k, v, dtype, spread=3.0):
    """Random logits with each draft made likely about half the time."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, k + 1, v, generator=g) * spread
    draft = torch.randint(0, v, (b, k), generator=g, dtype=torch.int32)
    if k:
        boost = torch.logsumexp(x[:, :k], 2) + 4 * torch.rand(
            b, k, generator=g) - 1.0
        x[:, :k].scatter_(2, draft.long()[..., None], boost[..., None])
    nv = torch.randint(0, k + 1, (b,), generator=g, dtype=torch.int32)
    nv[torch.rand(b, generator=g) < 0.5] = k
    u = torch.rand(b, k + 1, generator=g)
    return (x.to(dtype).to(DEV), draft.to(DEV), nv.to(DEV), u.to(DEV))


def _check(got, want):
    np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
    np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])
    assert got[0].dtype == got[1].dtype == torch.int32


def _np(*ts):
    return [None if t is None else t.cpu().numpy() for t in ts]


def _sampled(logits, draft, u, nv=None, t=1.0, k=None, p=None,
             row_start=None):
    """The operator and the oracle on the same inputs, compared. Numbers
    given as settings are rounded to fp32, as the drafter's are."""
    got = ops.verify_sampled(logits, draft, u, nv, t, k, p, row_start)
    as_np = [x.cpu().numpy() if torch.is_tensor(x) else
             np.float32(x) if isinstance(x, float) else x for x in (t, k, p)]
    d, n, uu, rs = _np(draft, nv, u, row_start)
    want = vo.verify_sampled(_f64(logits), d, uu, n, as_np[0],
                             0 if k is None else as_np[1],
                             1.0 if p is None else as_np[2], rs)
    _check(got, want)
    return got


SIZES = [(1, 0, 1), (3, 2, 1), (2, 1, 2), (5, 3, 7), (4, 5, 31), (2, 8, 257),
         (7, 4, 1000), (1, 16, 4099), (3, 2, 8192), (2, 3, 50021),
         (1, 0, 128256), (2, 32, 640)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("b,k,v", SIZES)
def test_sizes(b, k, v, dtype):
    logits, draft, nv, u = _case(b * 1000 + k + v, b, k, v, dtype)
    d, n = _np(draft, nv)
    _check(ops.verify_greedy(logits, draft, nv),
           vo.verify_greedy(_f64(logits), d, n))
    _sampled(logits, draft, u, nv)
    _sampled(logits, draft, u, None, 0.7)
    _sampled(logits, draft, u, nv, 1.3, p=0.9)
    _sampled(logits, draft, u, nv, 0.9, k=5)
    _sampled(logits, draft, u, nv, 1.1, k=max(1, v // 3), p=0.8)


def _probs_close(got: torch.Tensor, logits, t, k, p):
    """fp32 probabilities against the oracle's. The exponent (l - m) / T is
    formed in fp32: half a step of l - m, and 2 steps of the scaled product,
    act on the result relative to |l - m| / T; exp2 (2^-22), the scale by
    1 / Z and its rounding add 8 half steps. Results below the smallest
    normal number may be flushed."""
    x = _f64(logits).reshape(-1, logits.shape[-1])
    g = got.double().cpu().numpy().reshape(x.shape)
    per = len(x) // len(t)
    for i, row in enumerate(x):
        ti = float(np.float32(t[i // per]))
        want = vo.row_probs(row, ti, int(k[i // per]),
                            float(np.float32(p[i // per])))
        r = np.where(np.isnan(row), -np.inf, row)
        with np.errstate(invalid="ignore", over="ignore"):
            depth = np.where(want > 0, np.abs(r - r.max()) / ti, 0.0) \
                if ti > 0 else np.zeros_like(want)
        depth = np.nan_to_num(depth, nan=0.0)
        tol = 2.0 ** -24 * (3 * depth + 8) * want + 2.0 ** -126
        bad = np.abs(g[i] - want) > tol
        assert not bad.any(), (i, np.nonzero(bad)[0][:5], g[i][bad][:5],
                               want[bad][:5])
        assert (g[i][want == 0] == 0).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("b,k,v", SIZES)
def test_target_probs_sizes(b, k, v, dtype):
    logits, _, _, _ = _case(b + k + v, b, k, v, dtype)
    g = torch.Generator().manual_seed(v)
    t = 0.4 + torch.rand(b, generator=g)
    t[0] = 0.0 if b > 1 else t[0]
    kk = torch.randint(1, max(2, v), (b,), generator=g, dtype=torch.int32)
    pp = torch.rand(b, generator=g)
    none_k, none_p = np.zeros(b), np.ones(b)
    out = ops.target_probs(logits, t.to(DEV))
    assert out.shape == logits.shape and out.dtype == torch.float32
    _probs_close(out, logits, t, none_k, none_p)
    _probs_close(ops.target_probs(logits, t.to(DEV), kk.to(DEV)), logits, t,
                 kk, none_p)
    _probs_close(ops.target_probs(logits, t.to(DEV), top_p=pp.to(DEV)),
                 logits, t, none_k, pp)
    _probs_close(ops.target_probs(logits, t.to(DEV), kk.to(DEV), pp.to(DEV)),
                 logits, t, kk, pp)
    flat = ops.target_probs(logits[:, 0], 0.8, top_k=3)
    assert flat.shape == logits[:, 0].shape
    _probs_close(flat, logits[:, 0], [0.8] * b, [3] * b, none_p)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", [1, 5, 64, 1031, 40000])
def test_masks_and_special_values(dtype, v):
    """Rows of -inf, of the type's lowest value, with NaN, with +inf, with
    one token left, with -0 and +0 tied."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(v)
    rows = [torch.full((v,), NEG), torch.full((v,), low),
            torch.randn(v, generator=g), torch.randn(v, generator=g),
            torch.full((v,), NEG), torch.full((v,), float("nan")),
            torch.zeros(v), torch.full((v,), low), torch.randn(v, generator=g)]
    rows[2][::2] = float("nan")
    rows[3][v // 2:] = float("inf")
    rows[4][v - 1] = -3.0
    rows[6][::2] = -0.0
    rows[7][v // 3] = 1.0
    rows[8][: v // 2] = NEG
    x = torch.stack(rows).to(dtype)
    b = x.shape[0]
    logits = x[:, None].expand(b, 3, v).contiguous().to(DEV)
    draft = torch.tensor([[v - 1, v // 2]] * b, dtype=torch.int32,
                         device=DEV)
    u = torch.rand(b, 3, generator=g).to(DEV)
    u[::2, 0] = 0.0
    d, = _np(draft)
    _check(ops.verify_greedy(logits, draft), vo.verify_greedy(_f64(logits), d))
    for t in (1.0, 0.0, -1.0, 0.3, 50.0, float("inf"), 1e-30, 1e-44,
              float("nan")):
        _sampled(logits, draft, u, None, t)
        _sampled(logits, draft, u, None, t, k=2, p=0.6)
    for kk, pp in ((0, 1.0), (1, 1.0), (v // 2, 0.5), (v, 0.0), (-4, 2.0),
                   (2 ** 31 - 1, 1e-9)):
        _probs_close(ops.target_probs(logits, 0.9, kk, pp), logits, [0.9] * b,
                     [kk] * b, [pp] * b)


@pytest.mark.parametrize("p", [float("nan"), -1.0, 0.0, 1e-30, 0.5, 0.999999,
                               1.0, 7.0])
def test_top_p_borders(p):
    """Exact borders: equal weights (T = inf) of distinct values, so the
    kept mass is a multiple of 1/8; ties kept together."""
    vals = torch.tensor([3.0, 1.0, 2.0, 7.0, 6.0, 5.0, 4.0, 0.0])
    logits = vals.repeat(2, 2, 1).to(DEV)
    logits[1] = torch.tensor([1.0, 1, 2, 2, 2, 3, 3, 0])
    t = [float("inf")] * 2
    _probs_close(ops.target_probs(logits, float("inf"), top_p=p), logits, t,
                 [0, 0], [p, p])
    _probs_close(ops.target_probs(logits, float("inf"), top_k=4, top_p=p),
                 logits, t, [4, 4], [p, p])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", [33, 3001])
def test_acceptance_borders(dtype, v):
    """Uniforms next to the drafted token's probability, from both sides,
    and at it (a half): the 64-bit comparison decides."""
    b, k = 16, 3
    logits, draft, _, u = _case(v, b, k, v, dtype)
    x, d = _f64(logits), draft.cpu().numpy()
    un = u.cpu().numpy()
    for i in range(b):
        for j in range(k):
            p = vo.row_probs(x[i, j], np.float32(0.8))[d[i, j]]
            f = np.float32(p)
            lo = f if float(f) < p else np.nextafter(f, np.float32(0))
            un[i, j] = lo if (i + j) % 3 else np.nextafter(lo, np.float32(1))
    u = torch.from_numpy(un).to(DEV)
    s, c = _sampled(logits, draft, u, None, 0.8)
    assert c.max() > 1
    two = torch.full((1, 2, v), NEG, dtype=dtype, device=DEV)
    two[..., 3] = two[..., 20] = 1.5
    half = torch.tensor([[0.5, 0.5]], device=DEV)
    s, c = _sampled(two, torch.tensor([[3]], device=DEV), half)
    assert s.tolist() == [[20, -1]] and c.tolist() == [1]


def test_uniforms_at_the_ends():
    """u = 0, the largest fp32 below 1, 1 and NaN."""
    logits, draft, nv, _ = _case(3, 6, 2, 700, torch.float32)
    for val in (0.0, 1 - 2.0 ** -24, 1.0, float("nan")):
        u = torch.full((6, 3), val, device=DEV)
        _sampled(logits, draft, u, nv)
        _sampled(logits, draft, u, nv, 0.0)
        _sampled(logits, draft, u, nv, 0.5, p=0.7)


def test_counts_and_foreign_drafts():
    """num_valid below 0, 0, above K; drafts outside the vocabulary and -1
    inside the counted range."""
    b, k, v = 9, 4, 513
    logits, draft, _, u = _case(11, b, k, v, torch.bfloat16)
    draft[2, 1], draft[3, 0], draft[4, 2] = -1, v, 2 ** 31 - 1
    draft[5, 0] = -2 ** 31
    nv = torch.tensor([-1, 0, 4, 4, 9, 1, -2 ** 31, 2 ** 31 - 1, 3],
                      dtype=torch.int32, device=DEV)
    u[:, :k] *= 0.3
    s, c = _sampled(logits, draft, u, nv)
    assert s[0].tolist() == [-1] * 5 and c[0] == 0 and c[6] == 0
    _sampled(logits, draft, u, nv.long(), 0.8, k=20)
    d, n = _np(draft, nv)
    _check(ops.verify_greedy(logits, draft.long(), nv),
           vo.verify_greedy(_f64(logits), d, n))
    empty = ops.verify_greedy(logits[:0], draft[:0])
    assert empty[0].shape == (0, 5) and empty[1].shape == (0,)
    assert ops.target_probs(logits[:0]).shape == (0, 5, v)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", [17, 1027, 50021])
def test_packed_rows(dtype, v):
    """Packed rows; starts that leave the packed range count as rows without
    mass and are not read."""
    b, k = 5, 3
    logits, draft, nv, u = _case(v, b, k, v, dtype)
    keep = torch.arange(k + 1, device=DEV)[None] <= nv[:, None]
    packed = logits[keep]
    start = (torch.cumsum(nv + 1, 0) - (nv + 1)).to(torch.int32)
    got = _sampled(packed, draft, u, nv, 0.9, row_start=start)
    ref = ops.verify_sampled(logits, draft, u, nv, 0.9)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    _sampled(packed, draft, u, nv, 0.9, k=7, p=0.9, row_start=start.long())
    bad = start.clone()
    bad[0], bad[1], bad[2] = -1, packed.shape[0] - 1, 2 ** 31 - 1
    _sampled(packed, draft, u, None, 0.9, row_start=bad)
    s, c = ops.verify_greedy(packed[:0], draft, row_start=start)
    assert (s == -1).all() and (c == 0).all()
    probs = torch.softmax(packed.float(), 1)
    d, n, uu, rs = _np(draft, nv, u, bad)
    _check(ops.verify_probs(probs, draft, u, nv, row_start=bad),
           vo.verify_probs(_f64(probs), d, uu, n, row_start=rs))


@pytest.mark.parametrize("dtype", DT)
def test_strides_and_alignment(dtype):
    """Views: rows that start anywhere, a batch and position order of their
    own, repeated rows, one spare position, a column slice."""
    b, k, v = 3, 2, 1013
    logits, draft, nv, u = _case(5, b, k, v, dtype)
    want = ops.verify_sampled(logits, draft, u, nv, 0.9)
    wide = torch.full((k + 2, b, v + 13), 9.0, dtype=dtype, device=DEV)
    for off in (0, 1, 3, 5, 8):
        view = wide.transpose(0, 1)[:, :, off:off + v]
        view[:, :k + 1] = logits
        for got in (ops.verify_sampled(view, draft, u, nv, 0.9),
                    ops.verify_sampled(view, draft.t().contiguous().t(),
                                       u.t().contiguous().t(), nv, 0.9)):
            assert torch.equal(got[0], want[0])
            assert torch.equal(got[1], want[1])
        pr = ops.target_probs(view[:, :k + 1], 0.9, top_p=0.8)
        assert torch.equal(pr, ops.target_probs(logits, 0.9, top_p=0.8))
        # a row's sum is taken in groups that follow its alignment, so two
        # alignments agree to rounding: each is within the bound that
        # _probs_close derives, and so within twice that of the other
        pr = ops.target_probs(view[:, :k + 1], 0.9)
        _probs_close(pr, logits, [0.9] * b, [0] * b, [1.0] * b)
    same = logits[:1, :1].expand(b, k + 1, v)
    _sampled(same, draft, u, nv)
    odd = torch.empty(v * 4 + 7, dtype=dtype, device=DEV)
    packed = odd[3:3 + 4 * v].view(4, v)
    packed.copy_(logits.reshape(-1, v)[:4])
    _sampled(packed, draft[:1], u[:1],
             row_start=torch.ones(1, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("v", [3, 100, 2048, 33333])
@pytest.mark.parametrize("with_q", [False, True])
def test_probs(v, with_q):
    b, k = 6, 5
    logits, draft, nv, u = _case(v + with_q, b, k, v, torch.float32)
    p = torch.softmax(logits, 2)
    q = None
    if with_q:
        q = torch.softmax(logits[:, :k] * 0.7, 2)
        q[0] = p[0, :k]           # the same distribution: all accepted
        q[1, 0] = 0.0
        q[1, 0, draft[1, 0].long()] = 1.0
    p[2, 1] = 0.0                 # a row without mass
    p[3, 0, : v // 2] = float("nan")
    p[4, 0, 0] = -1.0
    p[5, 2, v - 1] = float("inf")
    d, n, uu, qq = _np(draft, nv, u, q)
    _check(ops.verify_probs(p, draft, u, nv, q),
           vo.verify_probs(p.cpu().numpy(), d, uu, n, qq))
    _check(ops.verify_probs(p, draft, u, None, q),
           vo.verify_probs(p.cpu().numpy(), d, uu, None, qq))
    for val in (0.0, 1.0, float("nan")):
        uc = torch.full_like(u, val)
        _check(ops.verify_probs(p, draft, uc, nv, q),
               vo.verify_probs(p.cpu().numpy(), d, uc.cpu().numpy(), n, qq))
    if with_q:  # strided views of both
        pv = torch.empty(k + 1, b, v + 3, device=DEV)[:, :, 1:1 + v]
        pv.copy_(p.transpose(0, 1))
        qv = torch.empty(k + 2, b, v + 1, device=DEV)[:k, :, :v]
        qv.copy_(q.transpose(0, 1))
        _check(ops.verify_probs(pv.transpose(0, 1), draft, u, nv,
                                qv.transpose(0, 1)),
               vo.verify_probs(p.cpu().numpy(), d, uu, n, qq))


def test_nothing_left_after_the_rejected_token():
    """All mass on a rejected draft: the draft itself is drawn."""
    logits = torch.full((1, 2, 40), NEG, device=DEV)
    logits[..., 7] = 2.0
    draft = torch.tensor([[7]], dtype=torch.int32, device=DEV)
    u = torch.tensor([[1.0, 0.5]], device=DEV)
    s, c = _sampled(logits, draft, u)
    assert s.tolist() == [[7, -1]] and c.tolist() == [1]
    s, c = ops.verify_probs(torch.softmax(logits, 2), draft, u)
    assert s.tolist() == [[7, -1]] and c.tolist() == [1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_beyond_32_bits(dtype):
    """Rows whose element offsets pass 2^31 (and 2^32 bytes)."""
    v = 1 << 16
    n = (1 << 31) // v + 3
    big = torch.empty(n, v, dtype=dtype, device=DEV)
    logits, draft, nv, u = _case(8, 1, 2, v, dtype)
    big[n - 3:] = logits[0]
    start = torch.tensor([n - 3], dtype=torch.int32, device=DEV)
    want = ops.verify_sampled(logits, draft, u, nv, 0.8, 50, 0.9)
    got = ops.verify_sampled(big, draft, u, nv, 0.8, 50, 0.9, start)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    far = torch.as_strided(big, (2, 3, v), ((n - 3) * v, v, 1))
    got = ops.verify_sampled(far, draft.expand(2, 2), u.expand(2, 3),
                             torch.tensor([-1, 2], device=DEV), 0.8)
    want = ops.verify_sampled(logits, draft, u, None, 0.8)
    assert torch.equal(got[0][1], want[0][0])
    got = ops.verify_greedy(far, draft.expand(2, 2),
                            torch.tensor([-1, 2], device=DEV))
    assert torch.equal(got[0][1], ops.verify_greedy(logits, draft)[0][0])


def test_streams_graphs_and_repeats():
    """The current stream is used; a captured call replays on new inputs;
    two graphs and eager calls on other streams do not disturb each other;
    repeated calls are bit-equal."""
    sets = [_case(s, 8, 4, 20011, torch.bfloat16) for s in range(3)]
    t = torch.full((8,), 0.8, device=DEV)
    want = [ops.verify_sampled(*x[:2], x[3], x[2], t, 50, 0.95)
            for x in sets]
    wantp = [ops.target_probs(x[0], t, top_p=0.9) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        outs = []
        for x, st in zip(sets, streams):
            with torch.cuda.stream(st):
                outs.append((ops.verify_sampled(*x[:2], x[3], x[2], t, 50,
                                                0.95),
                             ops.target_probs(x[0], t, top_p=0.9)))
        torch.cuda.synchronize()
        for (got, gp), w, wp in zip(outs, want, wantp):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
            assert torch.equal(gp, wp)
    bufs = [[y.clone() for y in sets[0]] for _ in range(2)]
    graphs = []
    for buf in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = (ops.verify_sampled(*buf[:2], buf[3], buf[2], t, 50, 0.95),
                   ops.verify_greedy(*buf[:2], buf[2]),
                   ops.target_probs(buf[0], t, top_p=0.9),
                   ops.verify_probs(ops.target_probs(buf[0], t, top_p=0.9),
                                    buf[1], buf[3], buf[2]))
        graphs.append((g, out))
    for i in range(4):
        for a, (buf, (g, out)) in enumerate(zip(bufs, graphs)):
            src = sets[(i + a) % 3]
            with torch.cuda.stream(streams[a]):
                for dst, y in zip(buf, src):
                    dst.copy_(y)
                g.replay()
        torch.cuda.synchronize()
        for a, (g, out) in enumerate(graphs):
            w = want[(i + a) % 3]
            x = sets[(i + a) % 3]
            assert torch.equal(out[0][0], w[0])
            assert torch.equal(out[0][1], w[1])
            gr = ops.verify_greedy(*x[:2], x[2])
            assert torch.equal(out[1][0], gr[0])
            assert torch.equal(out[2], wantp[(i + a) % 3])


def test_vocabularies_beyond_shared_memory():
    """Rows that do not fit a cluster's shared memory: refused where the row
    has to be held, verified where it is only read through."""
    v = 600_001
    logits, draft, nv, u = _case(2, 2, 1, v, torch.float32)
    _sampled(logits, draft, u, nv, 0.8)
    d, n = _np(draft, nv)
    _check(ops.verify_greedy(logits, draft, nv),
           vo.verify_greedy(_f64(logits), d, n))
    with pytest.raises(RuntimeError, match="beyond supported limits"):
        ops.target_probs(logits)
    with pytest.raises(RuntimeError, match="beyond supported limits"):
        ops.verify_sampled(logits, draft, u, nv, 0.8, top_p=0.9)
    half = logits.to(torch.bfloat16)
    _sampled(half, draft, u, nv, 0.8, p=0.9)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("fill", ["equal", "two", "near", "ramp", "flat"])
def test_filters_on_crowded_rows(fill, dtype):
    """Many values at or next to the borders: all equal, two values, values
    one step apart, a ramp far beyond the first bins, a wide flat row."""
    v = 20_011
    i = torch.arange(v, dtype=torch.float32)
    g = torch.Generator().manual_seed(5)
    row = {"equal": torch.full((v,), 2.5), "two": (i % 2) * 0.25,
           "near": 8.0 + (i % 701) * 2.0 ** -20,
           "ramp": -(i % 4999) * 0.03,
           "flat": torch.randn(v, generator=g) * 0.5}[fill]
    logits = row[torch.randperm(v, generator=g)].to(dtype)
    logits = logits.expand(6, 2, v).contiguous().to(DEV)
    t = torch.tensor([1.0, 0.3, 4.0, 60.0, 1.0, 0.05])
    k = torch.tensor([0, 7, 3000, 0, 19_000, 500], dtype=torch.int32)
    p = torch.tensor([0.9, 0.5, 0.97, 0.3, 1.0, 0.999])
    args = (t.to(DEV), k.to(DEV), p.to(DEV))
    # equal weights in the thousands: the fp32 sum's own rounding, 2^-24 for
    # each of at most 20 additions, comes on top of _probs_close's 8
    got = ops.target_probs(logits, *args)
    x = _f64(logits)
    for b in range(6):
        want = vo.row_probs(x[b, 0], float(t[b]), int(k[b]), float(p[b]))
        gb = got[b, 0].double().cpu().numpy()
        # weights below 2^-126 may be flushed; dropped tokens are 0
        assert (gb[want > 2.0 ** -125] > 0).all() and (gb[want == 0] == 0).all()
        depth = np.abs(x[b, 0] - x[b, 0].max()) / float(t[b])
        tol = 2.0 ** -24 * (3 * depth + 28) * want + 2.0 ** -126
        assert (np.abs(gb - want) <= tol).all()
    draft = torch.full((6, 1), 11, dtype=torch.int32, device=DEV)
    u = torch.rand(6, 2, generator=g).to(DEV)
    _sampled(logits, draft, u, None, *args)


def test_refusals_on_the_gpu():
    logits, draft, nv, u = _case(1, 2, 2, 64, torch.float32)
    with pytest.raises(ValueError, match="another device"):
        ops.verify_sampled(logits, draft.cpu(), u)
    with pytest.raises(ValueError, match="another device"):
        ops.verify_sampled(logits, draft, u.cpu())
    with pytest.raises(ValueError, match="another device"):
        ops.verify_greedy(logits, draft, nv.cpu())
    with pytest.raises(ValueError, match="another device"):
        ops.verify_sampled(logits, draft, u, temperature=torch.ones(2))
    with pytest.raises(ValueError, match="no backward pass"):
        ops.target_probs(logits.clone().requires_grad_())
    with torch.no_grad():
        ops.target_probs(logits.clone().requires_grad_())


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("enable_global", [False, True])
def test_decode_loop(sampled, enable_global):
    """propose -> target logits -> verify_and_propose over several steps
    equals the oracle drafter fed by the oracle verification, eagerly and
    from a captured graph."""
    k, b, s, v = 4, 6, 512, 60
    cfg = dict(k=k, max_pattern_len=8, max_occurrences=16, num_backoff=4,
               max_spec_factor=2.0, min_token_prob=0.05)
    data = wl.local_config(21, b=b, s=s, vocab=v, p_copy=0.8, span=(4, 40),
                           q_range=(100, 300))
    extra = dict(enable_global=True, global_capacity=1 << 12,
                 delta_capacity=1 << 9) if enable_global else {}
    d = SuffixGPUDrafter(device=DEV, **cfg, **extra)
    ora = so.SuffixDrafter(**cfg)
    tok = torch.from_numpy(data["token_ids"]).to(DEV)
    n = torch.from_numpy(data["num_tokens"]).to(DEV)
    tok_o, n_o = data["token_ids"].copy(), data["num_tokens"].copy()
    draft, nv = d.propose(n, tok)
    draft_o, nv_o = ora.propose(n_o, tok_o)
    g = torch.Generator().manual_seed(4)
    accepted = 0
    for _ in range(6):
        np.testing.assert_array_equal(draft.cpu().numpy(), draft_o)
        np.testing.assert_array_equal(nv.cpu().numpy(), nv_o)
        logits = torch.randn(b, k + 1, v, generator=g)
        idx = draft.cpu().long().clamp(min=0)[..., None]
        logits[:, :k].scatter_(2, idx, 5.0)
        u = torch.rand(b, k + 1, generator=g)
        kw = dict(uniforms=u.to(DEV), temperature=0.9, top_k=30,
                  top_p=0.95) if sampled else {}
        draft, nv, n, ids, cnt = d.verify_and_propose(
            logits.to(DEV), draft, nv, n, tok, **kw)
        if sampled:
            ids_o, cnt_o = vo.verify_sampled(
                logits.double().numpy(), draft_o, u.numpy(), nv_o,
                np.float32(0.9), 30,
                np.float32(0.95))
        else:
            ids_o, cnt_o = vo.verify_greedy(logits.double().numpy(), draft_o,
                                            nv_o)
        _check((ids, cnt), (ids_o, cnt_o))
        accepted += int(cnt_o.sum()) - b
        draft_o, nv_o, n_o = ora.propose_with_update(n_o, tok_o, ids_o, cnt_o)
        np.testing.assert_array_equal(n.cpu().numpy(), n_o)
        np.testing.assert_array_equal(tok.cpu().numpy(), tok_o)
    assert accepted > 0
