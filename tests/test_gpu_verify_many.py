"""Verification of more rows or requests than the GPU holds at once: rows
left out behind a rejection, requests decided by a second launch, clusters
that take several rows or requests, captured graphs. Small vocabularies,
against the 64-bit oracle."""

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


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _equal(got, want):
    np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
    np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])


def _case(seed, b, k, v, dtype, ragged):
    """Logits with likely drafts, inactive requests, temperatures of 0 among
    others; uniforms next to the drafts' probabilities for one request in
    two, so that many of them need sums in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(b, k + 1, v, generator=g) * 2.0).to(dtype)
    draft = torch.randint(0, v, (b, k), generator=g, dtype=torch.int32)
    if k:
        boost = torch.logsumexp(x[:, :k].float(), 2) + 4 * torch.rand(
            b, k, generator=g)
        x[:, :k].scatter_(2, draft.long()[..., None],
                          boost[..., None].to(dtype))
    nv = torch.randint(-1, k + 1, (b,), generator=g, dtype=torch.int32)
    nv[torch.rand(b, generator=g) < 0.6] = k
    t = 0.5 + torch.rand(b, generator=g)
    t[torch.rand(b, generator=g) < 0.1] = 0.0
    u = torch.rand(b, k + 1, generator=g)
    x64, d, un = _f64(x), draft.numpy(), u.numpy()
    for i in range(0, b, 2):
        if not t[i] > 0:
            continue
        for j in range(k):
            w = np.exp((x64[i, j] - x64[i, j].max()) / float(t[i]))
            p = w[d[i, j]] / w.sum()
            f = np.float32(p)
            below = f if float(f) < p else np.nextafter(f, np.float32(0))
            un[i, j] = below if (i // 2 + j) % 4 else np.nextafter(
                below, np.float32(1))
        # and the draw next to a border of the running sum
        p = np.cumsum(w / w.sum()) if k else np.cumsum(
            np.exp((x64[i, 0] - x64[i, 0].max()) / float(t[i])))
        un[i, k] = np.float32(p[v // 2] / p[-1])
    start = None
    rows = x
    if ragged:
        n = nv.clamp(min=-1) + 1
        start = (torch.cumsum(n, 0) - n).to(torch.int32)
        rows = x[torch.arange(k + 1)[None] <= nv[:, None]]
    dev = [None if y is None else y.to(DEV)
           for y in (rows, draft, nv, u, t, start)]
    return dev


def _fill_garbage():
    """Leaves freed blocks of the allocator's filled with -1 (NaN as Parts,
    -1 as counters): what the next workspaces are made of."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 22, 1 << 24):
        torch.full((n,), 255, dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("b,k,v", [(300, 16, 67), (129, 0, 1500),
                                   (90, 8, 801), (190, 5, 2049)])
def test_many_rows(b, k, v, ragged, dtype):
    """More rows than blocks (300 x 17, 90 x 9, 190 x 6) and more requests
    than the one-launch decision takes (300, 129, 190), greedy, sampled and
    filtered. What is left out depends on timing, the results do not."""
    rows, draft, nv, u, t, start = _case(b + k, b, k, v, dtype, ragged)
    r64 = _f64(rows)
    d, n, uu, tt = (y.cpu().numpy() for y in (draft, nv, u, t))
    s = None if start is None else start.cpu().numpy()
    want_g = vo.verify_greedy(r64, d, n, s)
    want_s = vo.verify_sampled(r64, d, uu, n, tt, row_start=s)
    want_k = vo.verify_sampled(r64, d, uu, n, tt, 40, np.float32(0.9), s)
    for _ in range(3):
        _fill_garbage()
        _equal(ops.verify_greedy(rows, draft, nv, start), want_g)
        _fill_garbage()
        _equal(ops.verify_sampled(rows, draft, u, nv, t, row_start=start),
               want_s)
        _fill_garbage()
        _equal(ops.verify_sampled(rows, draft, u, nv, t, 40, 0.9, start),
               want_k)


@pytest.mark.parametrize("v", [5003, 20011])
def test_rows_taken_in_turns(v):
    """Filtered rows by the hundred: clusters of several blocks take row
    after row, of changing kinds (top-p alone, top-k alone, both, greedy,
    without mass, all equal)."""
    b, k = 140, 4
    rows, draft, nv, u, t, _ = _case(7, b, k, v, torch.bfloat16, False)
    g = torch.Generator().manual_seed(1)
    rows[5::11] = float("-inf")
    rows[3::13, 1] = 0.5
    rows[4::17, :, 50:] = float("-inf")
    kk = torch.randint(0, 3, (b,), generator=g, dtype=torch.int32) * 30
    pp = torch.where(torch.rand(b, generator=g) < 0.6,
                     0.3 + 0.7 * torch.rand(b, generator=g), torch.ones(b))
    want = vo.verify_sampled(_f64(rows), draft.cpu().numpy(),
                             u.cpu().numpy(), nv.cpu().numpy(),
                             t.cpu().numpy(), kk.numpy(), pp.numpy())
    for _ in range(3):
        _fill_garbage()
        _equal(ops.verify_sampled(rows, draft, u, nv, t, kk.to(DEV),
                                  pp.to(DEV)), want)


@pytest.mark.parametrize("with_q", [False, True])
def test_many_requests_from_probabilities(with_q):
    b, k, v = 700, 3, 1201
    rows, draft, nv, u, t, _ = _case(11, b, k, v, torch.float32, False)
    p = torch.softmax(rows, 2)
    q = torch.softmax(rows[:, :k] * 0.8, 2) if with_q else None
    want = vo.verify_probs(_f64(p), draft.cpu().numpy(), u.cpu().numpy(),
                           nv.cpu().numpy(),
                           None if q is None else _f64(q))
    _equal(ops.verify_probs(p, draft, u, nv, q), want)


def test_captured_calls_with_many_rows():
    """Two captured graphs of every form, replayed in turn on two streams
    with new inputs: all outputs, counts among them, equal eager calls'."""
    b, k, v = 150, 5, 1009

    def forms(rows, draft, nv, u, t):
        p = ops.target_probs(rows, t)
        return [*ops.verify_greedy(rows, draft, nv),
                *ops.verify_sampled(rows, draft, u, nv, t),
                *ops.verify_sampled(rows, draft, u, nv, t, 30, 0.9),
                *ops.verify_probs(p, draft, u, nv),
                *ops.verify_probs(p, draft, u, nv, p[:, :k]), p]
    sets = [_case(s, b, k, v, torch.bfloat16, False)[:5] for s in range(3)]
    want = [forms(*x) for x in sets]
    bufs = [[y.clone() for y in sets[0]] for _ in range(2)]
    graphs = []
    for buf in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = forms(*buf)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(4):
        for a, (buf, (g, _)) in enumerate(zip(bufs, graphs)):
            streams[a].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[a]):
                for dst, y in zip(buf, sets[(i + a) % 3]):
                    dst.copy_(y)
                g.replay()
        torch.cuda.synchronize()
        for a, (_, out) in enumerate(graphs):
            for x, y in zip(out, want[(i + a) % 3]):
                assert torch.equal(x, y)


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("enable_global", [False, True])
def test_captured_decode_loop(sampled, enable_global):
    """verify_and_propose captured once and replayed, its counts and drafts
    fed back in place, equals the oracle drafter fed by the oracle
    verification."""
    k, b, s, v = 4, 6, 512, 60
    cfg = dict(k=k, max_pattern_len=8, max_occurrences=16, num_backoff=4,
               max_spec_factor=2.0, min_token_prob=0.05)
    data = wl.local_config(22, b=b, s=s, vocab=v, p_copy=0.8, span=(4, 40),
                           q_range=(100, 300))
    extra = dict(enable_global=True, global_capacity=1 << 12,
                 delta_capacity=1 << 9) if enable_global else {}
    d = SuffixGPUDrafter(device=DEV, **cfg, **extra)
    ora = so.SuffixDrafter(**cfg)
    tok = torch.from_numpy(data["token_ids"]).to(DEV)
    n = torch.from_numpy(data["num_tokens"]).to(DEV)
    tok_o, n_o = data["token_ids"].copy(), data["num_tokens"].copy()
    draft, nv = (x.clone() for x in d.propose(n, tok))
    draft_o, nv_o = ora.propose(n_o, tok_o)
    logits = torch.zeros(b, k + 1, v, device=DEV)
    u = torch.zeros(b, k + 1, device=DEV)
    kw = dict(uniforms=u, temperature=0.9, top_k=30,
              top_p=0.95) if sampled else {}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up on scratch copies
        d.verify_and_propose(logits, draft.clone(), nv.clone(), n.clone(),
                             tok.clone(), **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dr, nv2, n2, ids, cnt = d.verify_and_propose(logits, draft, nv, n,
                                                     tok, **kw)
        draft.copy_(dr)
        nv.copy_(nv2)
        n.copy_(n2)
    g = torch.Generator().manual_seed(4)
    accepted = 0
    for _ in range(6):
        lg = torch.randn(b, k + 1, v, generator=g)
        idx = torch.from_numpy(draft_o).long().clamp(min=0)[..., None]
        lg[:, :k].scatter_(2, idx, 5.0)
        un = torch.rand(b, k + 1, generator=g)
        logits.copy_(lg)
        u.copy_(un)
        graph.replay()
        torch.cuda.synchronize()
        if sampled:
            want = vo.verify_sampled(lg.double().numpy(), draft_o,
                                     un.numpy(), nv_o, np.float32(0.9), 30,
                                     np.float32(0.95))
        else:
            want = vo.verify_greedy(lg.double().numpy(), draft_o, nv_o)
        _equal((ids, cnt), want)
        accepted += int(want[1].sum()) - b
        draft_o, nv_o, n_o = ora.propose_with_update(n_o, tok_o, *want)
        np.testing.assert_array_equal(n.cpu().numpy(), n_o)
        np.testing.assert_array_equal(tok.cpu().numpy(), tok_o)
        np.testing.assert_array_equal(draft.cpu().numpy(), draft_o)
        np.testing.assert_array_equal(nv.cpu().numpy(), nv_o)
    assert accepted > 0
    del graph


def test_calls_from_several_threads():
    """Four threads, each on a stream of its own with a vocabulary of its
    own, whose rows need different amounts of shared memory."""
    import threading

    def forms(rows, draft, nv, u, t):
        return [*ops.verify_greedy(rows, draft, nv),
                *ops.verify_sampled(rows, draft, u, nv, t),
                *ops.verify_sampled(rows, draft, u, nv, t, 30, 0.9),
                ops.target_probs(rows, t),
                ops.target_probs(rows, t, top_p=0.9)]
    sets = [_case(v, 3, 2, v, torch.float32, False)[:5]
            for v in (9001, 90_001, 250_001, 40_001)]
    torch.cuda.synchronize()
    gate, got, errors = threading.Barrier(4, timeout=60), [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait()
                for _ in range(5):
                    got[i] = forms(*sets[i])
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # reported by the main thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    for x, out in zip(sets, got):
        for a, b in zip(forms(*x), out):
            assert torch.equal(a, b)
