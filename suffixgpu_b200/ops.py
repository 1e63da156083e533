"""Tensor-level wrappers of the sm_100a kernels.

These mirror the reference's operator layer (suffix_gpu/triton_kernels.py
and the op functions in expand.py / sa_search.py / suffix_array.py) with the
same argument meaning, shapes and return dtypes. Every op runs on CUDA
tensors only and raises otherwise: there is no CPU path.
"""

from __future__ import annotations

import torch

from suffixgpu_b200 import _lib
from suffixgpu_b200._lib import call, ptr, stream_of, torch_ops


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("suffixgpu_b200 ops need CUDA tensors "
                             f"(got a tensor on {t.device})")
        dev = t.device if dev is None else dev
    if dev is None:
        raise ValueError("no tensor given")
    return dev


def as_i32(t: torch.Tensor) -> torch.Tensor:
    t = t if t.dtype == torch.int32 else t.to(torch.int32)
    return t.contiguous()


def as_i64(t: torch.Tensor) -> torch.Tensor:
    t = t if t.dtype == torch.int64 else t.to(torch.int64)
    return t.contiguous()


def scatter_append(token_ids: torch.Tensor, base: torch.Tensor,
                   cnt: torch.Tensor | None,
                   sampled: torch.Tensor) -> torch.Tensor:
    """Append each row's valid sampled ids at its base offset, in place
    (triton_kernels.py:392-402). Returns the new counts [B] int32."""
    dev = require_cuda(token_ids, base, sampled)
    if token_ids.dtype != torch.int32 or token_ids.dim() != 2 \
            or token_ids.stride(1) != 1:
        raise ValueError("token_ids must be an int32 [B, S] tensor with "
                         "unit column stride")
    b, s = token_ids.shape
    base = as_i32(base)
    sampled = as_i32(sampled)
    cnt32 = None if cnt is None else as_i32(cnt)
    new = torch.empty(b, dtype=torch.int32, device=dev)
    call("sg_scatter_append", ptr(token_ids), token_ids.stride(0), b, s,
         ptr(base), ptr(cnt32), ptr(sampled), sampled.shape[1], ptr(new),
         stream_of(dev))
    return new


def match_back(src: torch.Tensor, pat: torch.Tensor,
               n_out: int) -> torch.Tensor:
    """match_back[b, i] = longest L with src[.., i-L:i] == tail_L
    (triton_kernels.py:259-281). src is [B, S] or a shared [N] buffer."""
    dev = require_cuda(src, pat)
    src = as_i32(src)
    pat = as_i32(pat)
    b, p = pat.shape
    out = torch.empty(b, n_out, dtype=torch.int32, device=dev)
    stride = src.stride(0) if src.dim() == 2 else 0
    n_src = src.shape[-1]
    call("sg_match_back", ptr(src), stride, n_src, ptr(pat), b, p, n_out,
         ptr(out), stream_of(dev))
    return out


def first_occurrences(mb: torch.Tensor, thr: torch.Tensor, c: int,
                      r: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Earliest r positions with mb >= per-candidate threshold
    (triton_kernels.py:362-389). Returns (pos [B*C, r] i64, count i64)."""
    dev = require_cuda(mb, thr)
    mb = as_i32(mb)
    thr = as_i64(thr)
    bc = thr.shape[0]
    pos = torch.empty(bc, r, dtype=torch.int64, device=dev)
    cnt = torch.empty(bc, dtype=torch.int64, device=dev)
    call("sg_first_occurrences", ptr(mb), mb.shape[1], ptr(thr), bc, c, r,
         ptr(pos), ptr(cnt), stream_of(dev))
    return pos, cnt


def expand_chain(cont: torch.Tensor, num_occ: torch.Tensor, k: int,
                 sentinel: int = -1, min_token_prob: float = 0.0,
                 cap: torch.Tensor | None = None,
                 weights: torch.Tensor | None = None,
                 alpha: float = 0.0):
    """Majority-vote chain expansion with fused scoring
    (suffix_gpu/expand.py:59-147). Returns (chain [B, k] int32, num_valid
    [B] i64, num_emit [B] i64, score [B] f32)."""
    if sentinel != -1:
        raise ValueError("only sentinel=-1 is supported")
    if weights is not None:
        raise NotImplementedError("weighted votes are not supported")
    dev = require_cuda(cont, num_occ)
    b, r, kk = cont.shape
    if kk < k:
        raise ValueError("cont has fewer than k columns")
    cont = as_i32(cont)
    if kk != k:
        cont = cont[:, :, :k].contiguous()
    num_occ = as_i64(num_occ)
    capc = None if cap is None else as_i64(cap)
    chain = torch.empty(b, k, dtype=torch.int32, device=dev)
    nv = torch.empty(b, dtype=torch.int64, device=dev)
    emit = torch.empty(b, dtype=torch.int64, device=dev)
    score = torch.empty(b, dtype=torch.float32, device=dev)
    call("sg_expand_chain", ptr(cont), b, r, k, ptr(num_occ), ptr(capc),
         float(min_token_prob), float(alpha), ptr(chain), ptr(nv),
         ptr(emit), ptr(score), stream_of(dev))
    return chain, nv, emit, score


# ---------------------------------------------------------------------------
# suffix array (suffix_gpu/suffix_array.py, sa_search.py)
# ---------------------------------------------------------------------------
_ws_cache: dict = {}


def _workspace(device: torch.device, nbytes: int, tag: str) -> torch.Tensor:
    """Cached per-device scratch buffer of at least nbytes."""
    key = (device.index, tag)
    buf = _ws_cache.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
        _ws_cache[key] = buf
    return buf


def build_suffix_array_into(tokens: torch.Tensor, out: torch.Tensor,
                            workspace: torch.Tensor | None = None,
                            stream: int | None = None) -> int:
    """Suffix array of the 1-D int32 tokens into the int32 `out` (same
    length). Returns the number of doubling rounds. Synchronises the
    stream it runs on (once per round)."""
    dev = require_cuda(tokens, out)
    tokens = as_i32(tokens.reshape(-1))
    n = tokens.numel()
    if out.dtype != torch.int32 or out.numel() < n or not out.is_contiguous():
        raise ValueError("out must be a contiguous int32 tensor of length n")
    L = _lib.lib()
    need = int(L.sg_suffix_array_workspace_size(n))
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(dev, need, "sa")
    rounds = _lib.c_int32(0)
    call("sg_build_suffix_array", ptr(tokens), n, ptr(out), ptr(workspace),
         workspace.numel(), _lib.ctypes.byref(rounds),
         stream if stream is not None else stream_of(dev))
    return int(rounds.value)


def append_suffix_array_into(tokens: torch.Tensor, out: torch.Tensor,
                             prev_sa: torch.Tensor, prev_n: int,
                             evicted: int, kept: int, prev_rounds: int,
                             workspace: torch.Tensor | None = None,
                             stream: int | None = None) -> int:
    """Suffix array of the 1-D int32 tokens into `out` from the suffix
    array of the previous snapshot (sg_suffix_array_append): tokens[:kept]
    must equal the previous snapshot's tokens[evicted:evicted + kept],
    prev_sa[:prev_n] be its suffix array and prev_rounds the rounds its
    build reported. Returns the new snapshot's rounds bound. Synchronises
    the stream it runs on."""
    dev = require_cuda(tokens, out, prev_sa)
    tokens = as_i32(tokens.reshape(-1))
    n = tokens.numel()
    if out.dtype != torch.int32 or out.numel() < n or not out.is_contiguous():
        raise ValueError("out must be a contiguous int32 tensor of length n")
    if (prev_sa.dtype != torch.int32 or not prev_sa.is_contiguous()
            or prev_sa.numel() < prev_n):
        raise ValueError("prev_sa must be a contiguous int32 tensor holding "
                         "prev_n entries")
    L = _lib.lib()
    need = int(L.sg_suffix_array_append_workspace_size(n))
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(dev, need, "sa_append")
    rounds = _lib.c_int32(0)
    call("sg_suffix_array_append", ptr(tokens), n, ptr(prev_sa), prev_n,
         evicted, kept, prev_rounds, ptr(out), ptr(workspace),
         workspace.numel(), _lib.ctypes.byref(rounds),
         stream if stream is not None else stream_of(dev))
    return int(rounds.value)


def build_suffix_array(tokens: torch.Tensor) -> torch.Tensor:
    """build_suffix_array (suffix_array.py:15-63): int64 start positions of
    the suffixes in lexicographic order."""
    dev = require_cuda(tokens)
    n = tokens.numel()
    out = torch.empty(n, dtype=torch.int32, device=dev)
    if n:
        build_suffix_array_into(tokens, out)
    return out.to(torch.int64)


def search_interval(sa: torch.Tensor, corpus: torch.Tensor,
                    pattern: torch.Tensor, pattern_len: torch.Tensor):
    """search_interval (sa_search.py:66-107): SA interval [start, end) of
    the suffixes starting with each pattern. Returns (start, end) int64."""
    dev = require_cuda(sa, corpus, pattern, pattern_len)
    sa = as_i32(sa)
    corpus = as_i32(corpus)
    pattern = as_i32(pattern)
    plen = as_i64(pattern_len)
    b, m = pattern.shape
    start = torch.empty(b, dtype=torch.int64, device=dev)
    end = torch.empty(b, dtype=torch.int64, device=dev)
    call("sg_sa_search", ptr(sa), ptr(corpus), sa.numel(), ptr(pattern), b,
         m, ptr(plen), ptr(start), ptr(end), stream_of(dev))
    return start, end


def suffix_match_backoff(sa, corpus, query, query_len, max_len: int, caps,
                         row_mask=None):
    """suffix_match_backoff (sa_search.py:110-163). Returns (match_len,
    start, end), each [B, C] int64."""
    dev = require_cuda(sa, corpus, query, query_len, caps)
    sa = as_i32(sa)
    corpus = as_i32(corpus)
    query = as_i32(query)
    qlen = as_i64(query_len)
    caps = as_i64(caps)
    b, q = query.shape
    c = caps.numel()
    out = [torch.empty(b, c, dtype=torch.int64, device=dev) for _ in range(3)]
    rm = None if row_mask is None else row_mask.to(torch.bool).contiguous()
    call("sg_suffix_match_backoff", ptr(sa), ptr(corpus), sa.numel(),
         ptr(query), b, q, ptr(qlen), max_len, ptr(caps), c, ptr(rm),
         ptr(out[0]), ptr(out[1]), ptr(out[2]), stream_of(dev))
    return out[0], out[1], out[2]


def longest_suffix_match(sa, corpus, query, query_len, max_len: int):
    """longest_suffix_match (sa_search.py:166-185)."""
    caps = torch.full((1,), max_len, dtype=torch.int64, device=sa.device)
    best, s, e = suffix_match_backoff(sa, corpus, query, query_len, max_len,
                                      caps)
    return best[:, 0], s[:, 0], e[:, 0]


# ---------------------------------------------------------------------------
# draft verification (no reference counterpart: the reference ends at the
# drafts and takes the sampled ids back)
# ---------------------------------------------------------------------------
_verify_ops: dict = {}


def _verify_op(name: str):
    """The operator's overload itself: the call skips the look-up by name
    and the choice of an overload (a microsecond or so)."""
    op = _verify_ops.get(name)
    if op is None:
        op = _verify_ops[name] = getattr(torch_ops(), name).default
    return op


def _setting(value, off):
    """(tensor, number) of a per-request setting: one of the two is used."""
    if value is None:
        return None, off
    if isinstance(value, torch.Tensor):
        return value, off
    return None, value


def verify_greedy(logits: torch.Tensor, draft: torch.Tensor,
                  num_valid: torch.Tensor | None = None,
                  row_start: torch.Tensor | None = None
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """Verification of drafts at temperature 0: each request's drafts are
    accepted while they equal the first largest token of their logits row,
    and the row after them gives one more token.

    logits: float32, bfloat16 or float16, [B, K + 1, V] (row j is the
    target's after draft j - 1; any strides over the first two dimensions),
    or packed [N, V] with row_start [B], request b's rows starting at
    row_start[b]. draft: [B, K] token ids. num_valid [B]: drafts of each
    request that count (None: K; negative: an inactive request, whose rows
    are not read). NaN logits count as masked (-inf).

    Returns (sampled [B, K + 1] int32, -1 past the count; count [B] int32),
    what propose_with_update takes as its sampled ids and their count. A
    row with nothing but -inf ends its request without a token."""
    return _verify_op("verify_greedy")(logits, draft, num_valid, row_start)


def verify_sampled(logits: torch.Tensor, draft: torch.Tensor,
                   uniforms: torch.Tensor,
                   num_valid: torch.Tensor | None = None,
                   temperature: torch.Tensor | float = 1.0,
                   top_k: torch.Tensor | int | None = None,
                   top_p: torch.Tensor | float | None = None,
                   row_start: torch.Tensor | None = None
                   ) -> tuple[torch.Tensor, torch.Tensor]:
    """Verification of drafts that keeps the target's distribution, from its
    logits and given random numbers; probabilities are not stored.

    Draft j (token x) is accepted while uniforms[b, j] < P_j(x); at the
    first rejection, or after the last draft, one more token is drawn with
    uniforms[b, K] by inverse CDF over token ids, from the row's P without
    the rejected token. uniforms: [B, K + 1] float32 in [0, 1).

    temperature, top_k, top_p: numbers or [B] tensors, floats rounded to
    float32. P is softmax(l / T) over the tokens that top_k (values >= the
    k-th largest, ties kept; 0 = off) and then top_p (the values >= t, t the
    largest one whose tokens >= t hold at least top_p of the kept mass;
    1 = off) leave. T <= 0 is greedy. Other arguments and the result as
    verify_greedy's. Decisions are those of 64-bit arithmetic on the logits
    as stored."""
    t, t_all = _setting(temperature, 1.0)
    k, k_all = _setting(top_k, 0)
    p, p_all = _setting(top_p, 1.0)
    return _verify_op("verify_sampled")(logits, draft, uniforms, num_valid, t,
                                        k, p, t_all, k_all, p_all, row_start)


def verify_probs(probs: torch.Tensor, draft: torch.Tensor,
                 uniforms: torch.Tensor,
                 num_valid: torch.Tensor | None = None,
                 draft_probs: torch.Tensor | None = None,
                 row_start: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """verify_sampled from float32 probabilities ([B, K + 1, V], or packed
    [N, V] with row_start). With draft_probs [B, K, V] float32, the
    distributions the drafts were drawn from, draft j is accepted while
    uniforms[b, j] * q_j(x) < p_j(x), and the token after a rejection is
    drawn from max(p - q, 0). Values that are negative or not finite count
    as 0; a row without mass ends its request without a token."""
    return _verify_op("verify_probs")(probs, draft, uniforms, num_valid,
                                      draft_probs, row_start)


def target_probs(logits: torch.Tensor,
                 temperature: torch.Tensor | float = 1.0,
                 top_k: torch.Tensor | int | None = None,
                 top_p: torch.Tensor | float | None = None) -> torch.Tensor:
    """The target's probabilities under verify_sampled's temperature, top_k
    and top_p, float32 in the shape of logits ([N, V] with [N] settings, or
    [B, J, V] with [B] settings; float32, bfloat16 or float16). Dropped
    tokens are exactly 0; a row of -inf gives zeros. No backward pass and no
    forward-mode derivative: inputs that ask for one are refused."""
    t, t_all = _setting(temperature, 1.0)
    k, k_all = _setting(top_k, 0)
    p, p_all = _setting(top_p, 1.0)
    return _verify_op("target_probs")(logits, t, k, p, t_all, k_all, p_all)
