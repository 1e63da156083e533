"""Edges of the draft-verification operators: borders deep in a row's tail,
infinite and very large temperatures, tiny uniforms, indices beyond 32
bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import verify_oracle as vo
from suffixgpu_b200 import ops

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy().astype(np.float64)


def _check(got, want):
    np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
    np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])


def _tuned_row(g, v, t, p, top_k, miss):
    """A row of one likely token and a tail around the border of top-p = p
    (about 200 values in 1/16 octave), with one token's weight chosen such
    that the mass ahead of the border's token misses p of the whole by
    `miss` (or passes it, if negative). Returns the row and how many of its
    tokens are kept, from sums of 80-bit floats."""
    c = 1 - float(p)
    depth = -np.log(c / 4600.0)
    x = t * -(depth - 2 + 7 * torch.rand(v, generator=g))
    x[77], x[78] = 0.0, t * np.log(2e-6)
    tt = np.longdouble(np.float32(t))

    def border(x):
        s = np.sort(x.numpy())[::-1].astype(np.longdouble)
        s = s[:top_k] if top_k else s
        cum = np.cumsum(np.exp(s / tt))
        return cum, np.longdouble(p) * cum[-1]
    cum, need = border(x)
    m = int((cum < need).sum())  # cum[m - 1] < need <= cum[m]
    more = float(need - cum[m - 1] - miss) / c
    x[78] = t * np.log(2e-6 + more)
    cum, need = border(x)
    assert cum[m - 2] < need < cum[m]
    gap = float(need - cum[m - 1])
    assert miss / 2 < gap < 2 * miss or 2 * miss < gap < miss / 2
    return x, m + (gap > 0)


@pytest.mark.parametrize("top_k", [0, 15_000])
def test_top_p_borders_deep_in_the_tail(top_k):
    """top-p 4e-6 below 1 where the border's tokens weigh 2^-30 of the
    largest, and the mass ahead of one of them is 2e-13 more or less than
    top-p's share.

    64-bit sums of the row tell those apart: they are off by at most 2^-46
    (1.4e-14) of it, 40 * 2^-53 for the weights (their exponents' rounding,
    24 at a mean depth of 17 octaves, the series and 8 roundings) and 65 *
    2^-53 for the additions on a weight's way; and top-p's share the same."""
    n, v, t = 48, 32_003, 0.2
    p = np.float32(1 - 4e-6)
    g = torch.Generator().manual_seed(9 + top_k)
    rows, want = zip(*[_tuned_row(g, v, t, p, top_k,
                                  2e-13 if i % 2 else -2e-13)
                       for i in range(n)])
    logits = torch.stack(rows).to(DEV)
    out = ops.target_probs(logits, t, top_k or None, float(p))
    low = torch.where(out > 0, logits, float("inf")).amin(1)
    assert ((logits >= low[:, None]) == (out > 0)).all()
    assert (out > 0).sum(1).tolist() == list(want)


def test_indices_beyond_32_bits():
    """64-bit drafts, counts, row starts and top-k beyond 32 bits keep their
    meaning: a draft outside the vocabulary, all (or no) drafts, a row
    outside the packed ones, no limit."""
    b, k, v = 6, 2, 300
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(b, k + 1, v, generator=g)
    far = 2 ** 32
    draft = torch.randint(0, v, (b, k), generator=g)
    logits[:, :k].scatter_(2, draft[..., None], 9.0)
    u = torch.rand(b, k + 1, generator=g) * 0.5
    x64, un = logits.double().numpy(), u.numpy()
    x, u = logits.to(DEV), u.to(DEV)
    foreign = draft.clone()
    foreign[0, 0] += far
    foreign[1, 1] += 2 * far
    foreign[2, 0] -= far
    foreign[3, 1] = 2 ** 63 - 1
    foreign[4, 0] = -2 ** 63
    _check(ops.verify_greedy(x, foreign.to(DEV)),
           vo.verify_greedy(x64, foreign.numpy()))
    _check(ops.verify_sampled(x, foreign.to(DEV), u),
           vo.verify_sampled(x64, foreign.numpy(), un))
    p = torch.softmax(x, 2)
    _check(ops.verify_probs(p, foreign.to(DEV), u),
           vo.verify_probs(_f64(p), foreign.numpy(), un))
    nv = torch.tensor([far, -far, 1 - far, far + 1, 2 ** 63 - 1, -2 ** 63])
    _check(ops.verify_greedy(x, draft.to(DEV), nv.to(DEV)),
           vo.verify_greedy(x64, draft.numpy(), nv.numpy()))
    packed = x.reshape(-1, v)
    start = torch.tensor([0, far, 3 - far, far + 3, 2 ** 63 - 1, -2 ** 63])
    want = vo.verify_sampled(x64.reshape(-1, v), draft.numpy(), un,
                             row_start=start.numpy())
    assert want[1].tolist()[1:] == [0] * 5
    _check(ops.verify_sampled(packed, draft.to(DEV), u,
                              row_start=start.to(DEV)), want)
    kk = torch.tensor([far + 1, far, 2 ** 63 - 1, -2 ** 63, 1 - far, 2])
    _check(ops.verify_sampled(x, draft.to(DEV), u, None, 3.0, kk.to(DEV)),
           vo.verify_sampled(x64, draft.numpy(), un, None, 3.0,
                             kk.numpy()))
    out = ops.target_probs(x, 3.0, kk.to(DEV))
    assert (out > 0).sum(2).tolist() == [[v] * 3] * 5 + [[2] * 3]
    # strided, as the 32-bit ones may be
    wide = torch.stack([foreign, draft], 2).to(DEV)[:, :, 0]
    _check(ops.verify_greedy(x, wide),
           vo.verify_greedy(x64, foreign.numpy()))


def _special_rows(v, dtype):
    """Rows with infinite, NaN and masked entries, and one of plain ones."""
    g = torch.Generator().manual_seed(v)
    x = torch.randn(7, v, generator=g)
    x[0, v // 2:] = float("inf")
    x[1, v - 1] = float("inf")
    x[2, ::2] = float("inf")
    x[2, 1::2] = float("-inf")
    x[3, ::3] = float("nan")
    x[3, 0] = float("inf")
    x[4, :] = float("inf")
    x[5, 1:] = float("-inf")
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("v", [2, 9, 1031, 40000])
def test_infinite_temperature_and_logits(v, dtype):
    """T = +inf on rows with +inf entries: those share the mass, with
    and without filters, in every form. A probability is off by ex2's 2^-22
    at most, or by the roundings of 1 / Z and of the product."""
    x = _special_rows(v, dtype)
    logits = x[:, None].repeat(1, 2, 1).to(DEV)
    b, inf = x.shape[0], float("inf")
    off = torch.zeros(b, dtype=torch.int32, device=DEV)
    for kk, pp in ((0, 1.0), (off, 1.0), (v // 2, 1.0), (0, 0.75),
                   (v // 2, 0.5)):
        out = ops.target_probs(logits, inf, kk, pp).cpu().numpy()
        k = 0 if torch.is_tensor(kk) else kk
        for i in range(b):
            want = vo.row_probs(_f64(x[i]), inf, k, pp)
            for j in range(2):
                np.testing.assert_allclose(out[i, j], want, rtol=2.0 ** -22 + 2.0 ** -23,
                                           atol=0)
    draft = torch.tensor([[v // 2]] * b, dtype=torch.int32)
    u = torch.rand(b, 2, generator=torch.Generator().manual_seed(1))
    for kk, pp in ((0, 1.0), (3, 0.6)):
        _check(ops.verify_sampled(logits, draft.to(DEV), u.to(DEV), None, inf,
                                  kk, pp),
               vo.verify_sampled(_f64(logits), draft.numpy(), u.numpy(),
                                 None, inf, kk, np.float32(pp)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [5, 1009, 20011])
@pytest.mark.parametrize("t", [1e20, 1e24, 1e29, 2e30, 1e37, 3e38,
                               float("inf")])
def test_very_large_temperatures(t, v, dtype):
    """Temperatures up to fp32's largest number and +inf, on logits as large:
    spread out like the temperature, and near both ends of the type's range,
    where l - m passes fp32's.

    A probability's error in half steps (2^-24): 5 for each unit of depth
    (l - m) / T (l - m and the product one each, the scale 2.8 where it is
    below the smallest normal number), 4 for ex2, 2 for 1 / Z and the
    product, 20 additions, 2 for the scale's other rounding in the sum."""
    g = torch.Generator().manual_seed(v)
    big = torch.finfo(dtype).max
    size = min(t, big / 8)
    x = torch.randn(4, v, generator=g)
    x = (x * size).clamp(-big, big)
    ends = torch.rand(v, generator=g)
    x[1] = torch.where(ends < 0.3, big, torch.where(ends < 0.6, -big, 0.0))
    x[2] = torch.where(ends < 0.5, -big, x[2])
    x[2, 0] = big
    x[3] = torch.where(ends < 0.5, float("-inf"), x[3])
    x = x.to(dtype)
    x = torch.where(torch.isinf(x) & (x > 0), big, x)
    logits = x[:, None].repeat(1, 2, 1).to(DEV)
    x64 = _f64(x)
    tt = float(np.float32(t))
    for k, p in ((0, 1.0), (v // 2, 0.7)):
        out = _f64(ops.target_probs(logits, t, k, p))
        for i in range(4):
            want = vo.row_probs(x64[i], tt, k, float(np.float32(p)))
            m = x64[i].max()
            depth = np.where(want > 0, m - x64[i], 0.0) / tt
            tol = 2.0 ** -24 * (5 * depth + 28) * want
            assert (np.abs(out[i] - want) <= tol + 2.0 ** -126).all()
            assert (out[i][:, want == 0] == 0).all()
    draft = torch.randint(0, v, (4, 1), generator=g)
    u = torch.rand(4, 2, generator=g)
    for k, p in ((0, 1.0), (v // 2, 0.7)):
        _check(ops.verify_sampled(logits, draft.to(DEV), u.to(DEV), None, t,
                                  k, p),
               vo.verify_sampled(_f64(logits), draft.numpy(), u.numpy(),
                                 None, np.float32(t), k, np.float32(p)))


@pytest.mark.parametrize("b", [1, 160])
@pytest.mark.parametrize("v", [3, 2049])
def test_tiny_uniforms_and_probabilities(v, b):
    """Uniforms and drafted tokens' probabilities below the smallest normal
    fp32 number, next to one another: u < P(x) as 64 bits have it. Few
    requests and (b x 4 rows) more than one launch decides."""
    deep = torch.tensor([-86.5, -87.0, -87.5, -88.5, -90.0, -95.0, -102.0])
    g = torch.Generator().manual_seed(b + v)
    x = torch.full((b, 4, v), float("-inf"))
    x[..., 1] = 0.0
    d = deep[torch.randint(0, 7, (b, 3), generator=g)]
    d[:, 0] = -90.0
    x[:, :3, 0] = d
    u = torch.exp(d.double()) * torch.tensor([0.25, 0.5, 0.9, 1.1, 2.0])[
        torch.randint(0, 5, (b, 3), generator=g)]
    u = torch.cat([u.float(), torch.rand(b, 1, generator=g)], 1)
    u[:, 0] = 5e-40
    draft = torch.zeros(b, 3, dtype=torch.int32)
    want = vo.verify_sampled(x.double().numpy(), draft.numpy(), u.numpy())
    assert (want[1] > 1).all()
    _check(ops.verify_sampled(x.to(DEV), draft.to(DEV), u.to(DEV)), want)
    _check(ops.verify_sampled(x.to(DEV), draft.to(DEV), u.to(DEV), None, 1.0,
                              0, 1 - 2.0 ** -24),
           vo.verify_sampled(x.double().numpy(), draft.numpy(), u.numpy(),
                             None, 1.0, 0, np.float32(1 - 2.0 ** -24)))


def test_largest_vocabulary_held_on_chip():
    """380 thousand fp32 logits a row, with filters and without; 420 thousand
    are refused."""
    v = 380_000
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 1, v, generator=g) * 3
    draft = torch.empty(2, 0, dtype=torch.int32)
    u = torch.rand(2, 1, generator=g)
    _check(ops.verify_sampled(x.to(DEV), draft.to(DEV), u.to(DEV), None, 0.9,
                              40, 0.9),
           vo.verify_sampled(x.double().numpy(), draft.numpy(), u.numpy(),
                             None, np.float32(0.9), 40, np.float32(0.9)))
    out = ops.target_probs(x.to(DEV), 0.9)
    want = torch.softmax(x.double() / float(np.float32(0.9)), 2)
    # as _probs_close in the sizes' tests, with 20 additions more: depth is
    # at most 2 * 5.5 * 3 / 0.9 < 40
    np.testing.assert_allclose(out.double().cpu(), want,
                               rtol=2.0 ** -24 * (3 * 40 + 28))
    far = torch.zeros(1, 420_000, device=DEV)
    for k in (0, 40):
        with pytest.raises(RuntimeError, match="beyond supported limits"):
            ops.target_probs(far, 0.9, k)


@pytest.mark.parametrize("b,k", [(1, 0), (1, 1), (5, 3), (300, 2),
                                 (70_000, 5)])
def test_64_bit_indices_of_any_layout(b, k):
    """Contiguous, transposed, sliced and expanded 64-bit tensors give what
    the 32-bit ones do (70 thousand requests: more elements than threads)."""
    v = 5
    g = torch.Generator().manual_seed(b)
    x = torch.randn(b, k + 1, v, generator=g).to(DEV)
    draft = torch.randint(-1, v + 1, (b, k), generator=g).to(DEV)
    nv = torch.randint(-1, k + 2, (b,), generator=g).to(DEV)
    kk = torch.randint(0, v + 2, (b,), generator=g).to(DEV)
    u = torch.rand(b, k + 1, generator=g).to(DEV)

    def both(draft, nv, kk):
        a = ops.verify_sampled(x, draft, u, nv, 0.8, kk)
        c = ops.verify_sampled(x, draft.int().contiguous(), u,
                               nv.int().contiguous(), 0.8,
                               kk.int().contiguous())
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    both(draft, nv, kk)
    both(draft.t().contiguous().t(), torch.stack([nv, kk], 1)[:, 0],
         torch.stack([nv, kk], 1)[:, 1])
    both(torch.cat([draft, draft], 1)[:, k:], nv[:1].expand(b),
         kk[:1].expand(b))
    both(draft[:1].expand(b, k), nv, kk)
