"""Draft verification without a GPU: the oracle on hand-computed cases, and
the operators' refusals, which all come before any CUDA call."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import verify_oracle as vo
from suffixgpu_b200 import _lib, ops

NEG = -np.inf


def test_row_probs_by_hand():
    x = np.log(np.array([1.0, 2.0, 4.0, 1.0]))
    np.testing.assert_allclose(vo.row_probs(x, 1.0), [1/8, 2/8, 4/8, 1/8])
    np.testing.assert_allclose(vo.row_probs(x, 0.5),
                               np.array([1, 4, 16, 1]) / 22)
    # ties at the k-th value stay together
    np.testing.assert_allclose(vo.row_probs(x, 1.0, k=3),
                               [1/8, 2/8, 4/8, 1/8])
    np.testing.assert_allclose(vo.row_probs(x, 1.0, k=2), [0, 1/3, 2/3, 0])
    # 4/8 >= 0.5 alone; 6/8 >= 0.6; the two 1s together reach 0.8
    np.testing.assert_allclose(vo.row_probs(x, 1.0, p=0.4), [0, 0, 1, 0])
    np.testing.assert_allclose(vo.row_probs(x, 1.0, p=0.6), [0, 1/3, 2/3, 0])
    np.testing.assert_allclose(vo.row_probs(x, 1.0, p=0.8),
                               [1/8, 2/8, 4/8, 1/8])
    np.testing.assert_allclose(vo.row_probs(x, 1.0, p=0.0), [0, 0, 1, 0])
    # top-p is taken of what top-k leaves: 4/6 >= 0.66
    np.testing.assert_allclose(vo.row_probs(x, 1.0, k=2, p=0.66),
                               [0, 0, 1, 0])
    np.testing.assert_allclose(vo.row_probs([0, 3, 3], 0.0), [0, 1, 0])
    assert vo.row_probs([NEG, np.nan], 1.0).sum() == 0
    np.testing.assert_allclose(vo.row_probs([np.inf, 0, np.inf], 1.0),
                               [0.5, 0, 0.5])
    np.testing.assert_allclose(vo.row_probs([1, NEG, 5], np.inf),
                               [0.5, 0, 0.5])


def test_draw_by_hand():
    r = [0.0, 0.25, 0.0, 0.5, 0.25]
    assert [vo.draw(r, u) for u in (0.0, 0.2, 0.25, 0.7, 0.75, 0.99, 1.0,
                                    np.nan)] == [1, 1, 3, 3, 4, 4, 4, 4]
    assert vo.draw([0.0, 0.0], 0.5) == -1


def test_verification_by_hand():
    p = np.array([[[0.5, 0.5, 0.0], [0.1, 0.2, 0.7], [0.0, 0.0, 1.0]]])
    lg = np.log(p + 1e-300)
    u = np.array([[0.4, 0.19, 0.5]])
    s, c = vo.verify_probs(p, [[0, 1]], u)
    assert s.tolist() == [[0, 1, 2]] and c.tolist() == [3]
    s, c = vo.verify_sampled(lg, [[0, 1]], u)
    assert s.tolist() == [[0, 1, 2]] and c.tolist() == [3]
    u = np.array([[0.4, 0.21, 0.1]])  # second draft rejected
    s, c = vo.verify_probs(p, [[0, 1]], u)
    # residual 0.1, 0, 0.7: 0.1 * 0.8 < 0.1
    assert s.tolist() == [[0, 0, -1]] and c.tolist() == [2]
    u = np.array([[0.5, 0.0, 0.9]])  # u = p is a rejection
    s, c = vo.verify_probs(p, [[0, 1]], u)
    assert s.tolist() == [[1, -1, -1]] and c.tolist() == [1]
    # with draft probabilities: residual max(p - q, 0) = (0, 0, 0.6)
    q = np.array([[[0.5, 0.5, 0.0], [0.5, 0.4, 0.1]]])
    s, c = vo.verify_probs(p, [[0, 1]], np.array([[0.9, 0.6, 0.0]]),
                           draft_probs=q)
    assert s.tolist() == [[0, 2, -1]] and c.tolist() == [2]
    # inactive, no drafts, a draft outside the vocabulary
    p4 = np.repeat(p, 3, axis=0)
    s, c = vo.verify_probs(p4, [[0, 1], [0, 1], [7, 1]],
                           np.full((3, 3), 0.3), num_valid=[-1, 0, 2])
    assert s.tolist() == [[-1] * 3, [0, -1, -1], [0, -1, -1]]
    assert c.tolist() == [0, 1, 1]


def test_accepted_and_drawn_tokens_follow_the_target():
    """Averaged over uniforms on a grid, the first emitted token has the
    target's distribution whatever was drafted."""
    p = np.array([0.15, 0.35, 0.5])
    n = 400
    g = (np.arange(n) + 0.5) / n
    for x in range(3):
        hist = np.zeros(3)
        for u0 in g[::20]:
            for u1 in g[::4]:
                s, _ = vo.verify_probs(np.stack([p, p])[None], [[x]],
                                       np.array([[u0, u1]]))
                hist[s[0, 0]] += 1
        np.testing.assert_allclose(hist / hist.sum(), p, atol=0.03)


def _args(b=2, k=2, v=9, dtype=torch.float32):
    return (torch.zeros(b, k + 1, v, dtype=dtype),
            torch.zeros(b, k, dtype=torch.int32), torch.rand(b, k + 1))


@pytest.mark.parametrize("change,match", [
    (lambda a: a, "CUDA tensors"),
    (lambda a: (a[0].double(), a[1], a[2]), "float32, bfloat16 or float16"),
    (lambda a: (a[0][:, :2], a[1], a[2]), "every position"),
    (lambda a: (a[0][:1], a[1], a[2]), "every position"),
    (lambda a: (a[0][0], a[1], a[2]), r"\[B, K \+ 1, V\]"),
    (lambda a: (a[0][..., :0], a[1], a[2]), "empty vocabulary"),
    (lambda a: (a[0].transpose(1, 2).contiguous().transpose(1, 2), a[1],
                a[2]), "unit stride"),
    (lambda a: (a[0], a[1].float(), a[2]), "draft must be an integer"),
    (lambda a: (a[0], a[1][0], a[2]), r"draft must be a \[B, K\]"),
    (lambda a: (a[0], a[1], a[2][:, :2]), "uniforms"),
    (lambda a: (a[0], a[1], a[2].double()), "uniforms"),
])
def test_refused_arguments(change, match):
    logits, draft, u = change(_args())
    with pytest.raises(ValueError, match=match):
        ops.verify_sampled(logits, draft, u)
    if "uniforms" not in match:
        with pytest.raises(ValueError, match=match):
            ops.verify_greedy(logits, draft)
        if "float16" not in match:
            with pytest.raises(ValueError, match=match):
                ops.verify_probs(logits, draft, u)


@pytest.mark.parametrize("kw,match", [
    (dict(num_valid=torch.zeros(3, dtype=torch.int32)), "num_valid"),
    (dict(num_valid=torch.zeros(2)), "num_valid must be an integer"),
    (dict(row_start=torch.zeros(2, dtype=torch.int32)), r"\[N, V\]"),
    (dict(temperature=torch.ones(3)), "temperature must be a number or"),
    (dict(temperature=torch.ones(2, dtype=torch.int32)), "floating"),
    (dict(top_k=torch.ones(2)), "top_k must be an integer"),
    (dict(top_p=torch.ones(2, 1)), "top_p must be a number or"),
])
def test_refused_settings(kw, match):
    logits, draft, u = _args()
    with pytest.raises(ValueError, match=match):
        ops.verify_sampled(logits, draft, u, **kw)


def test_refused_probs_and_target_probs():
    logits, draft, u = _args()
    with pytest.raises(ValueError, match="probs must be a float32"):
        ops.verify_probs(logits.to(torch.bfloat16), draft, u)
    with pytest.raises(ValueError, match="draft_probs must be a float32"):
        ops.verify_probs(logits, draft, u, draft_probs=logits[:, :2].half())
    with pytest.raises(ValueError, match="every position"):
        ops.verify_probs(logits, draft, u, draft_probs=logits[:, :1])
    with pytest.raises(ValueError, match="differ in vocabulary"):
        ops.verify_probs(logits, draft, u, draft_probs=logits[:, :2, :5])
    with pytest.raises(ValueError, match=r"\[N, V\] or \[B, J, V\]"):
        ops.target_probs(logits[0, 0])
    with pytest.raises(ValueError, match="no backward pass"):
        ops.target_probs(logits[0].clone().requires_grad_())
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.target_probs(logits[0])


def test_refused_at_the_c_abi():
    """Bad row sets, missing pointers and short workspaces come back as
    status codes; an empty batch is nothing to do."""
    L = _lib.lib()
    assert ctypes.sizeof(_lib.Rows) == 64
    assert _lib.Rows.vocab.offset == 24
    assert ctypes.sizeof(_lib.Sampling) == 40
    one = 4096  # never dereferenced: every call below is refused
    ok = dict(data=one, dtype=0, batch=2, positions=3, vocab=9, stride_b=27,
              stride_j=9)

    def greedy(ws=one, wsb=1 << 20, draft=one, out=one, cnt=one, **kw):
        r = _lib.Rows(**{**ok, **kw})
        return L.sg_verify_greedy(ctypes.byref(r), draft, None, out, cnt, ws,
                                  wsb, None)
    need = L.sg_verify_workspace_size(2, 3)
    assert need > 0 and L.sg_verify_workspace_size(0, 3) == 0
    assert greedy(batch=0) == 0
    assert greedy(batch=-1) == 1 and greedy(positions=0) == 1
    assert greedy(dtype=3) == 1 and greedy(dtype=-1) == 1
    assert greedy(vocab=0) == 1 and greedy(vocab=1 << 31) == 1
    assert greedy(data=None) == 1 and greedy(stride_b=-1) == 1
    assert greedy(row_start=one, n_rows=-1) == 1
    assert greedy(row_start=one, n_rows=4, data=None) == 1
    assert greedy(draft=None) == 1 and greedy(out=None) == 1
    assert greedy(cnt=None) == 1
    assert greedy(ws=None) == 2 and greedy(wsb=need - 1) == 2
    assert greedy(ws=one + 8) == 2
    assert L.sg_verify_greedy(None, one, None, one, one, one, 99, None) == 1
    r = _lib.Rows(**ok)
    s = _lib.Sampling(temperature_all=1.0, top_p_all=1.0)
    assert L.sg_verify_sampled(ctypes.byref(r), ctypes.byref(s), one, None,
                               None, one, one, one, 1 << 20, None) == 1
    assert L.sg_verify_sampled(ctypes.byref(r), None, one, None, one, one,
                               one, one, 1 << 20, None) == 1
    assert L.sg_verify_probs(ctypes.byref(r), ctypes.byref(r), one, None,
                             one, one, one, None) == 1  # q has K positions
    assert L.sg_verify_probs(ctypes.byref(r), None, one, None, None, one,
                             one, None) == 1
    half = _lib.Rows(**{**ok, "dtype": 1})
    assert L.sg_verify_probs(ctypes.byref(half), None, one, None, one, one,
                             one, None) == 4
    assert L.sg_target_probs(ctypes.byref(r), ctypes.byref(s), None,
                             None) == 1
    assert L.sg_target_probs(ctypes.byref(r), None, one, None) == 1
    packed = _lib.Rows(**{**ok, "row_start": one, "n_rows": 6})
    assert L.sg_target_probs(ctypes.byref(packed), ctypes.byref(s), one,
                             None) == 1


def test_drafter_verify_refuses_settings_without_uniforms():
    from suffixgpu_b200 import SuffixGPUDrafter
    d = object.__new__(SuffixGPUDrafter)
    logits, draft, _ = _args()
    with pytest.raises(ValueError, match="need uniforms"):
        d.verify(logits, draft, temperature=0.7)
    with pytest.raises(ValueError, match="CUDA tensors"):
        d.verify(logits, draft)


def test_refused_packed_rows_beyond_32_bit_starts():
    """Row starts are 32-bit numbers; more packed rows than those reach are
    refused, not cut."""
    draft = torch.zeros(2, 1, dtype=torch.int32)
    start = torch.zeros(2, dtype=torch.int64)
    rows = torch.zeros(1, 4).expand(2 ** 31, 4)
    with pytest.raises(ValueError, match="2\\^31 packed rows"):
        ops.verify_greedy(rows, draft, row_start=start)
    with pytest.raises(ValueError, match="2\\^31 packed rows"):
        ops.verify_probs(rows, draft, torch.rand(2, 2), row_start=start)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.verify_greedy(rows[1:], draft, row_start=start)


def test_target_probs_refuses_every_kind_of_derivative():
    """Forward mode, function transforms and settings that need a gradient,
    none of which the operator has, are refused like a backward pass."""
    import torch.autograd.forward_ad as fwad
    x = torch.randn(2, 9)
    t = torch.ones(2)
    match = "no backward pass"
    with fwad.dual_level():
        with pytest.raises(ValueError, match=match):
            ops.target_probs(fwad.make_dual(x, x))
        with pytest.raises(ValueError, match=match):
            ops.target_probs(x, fwad.make_dual(t, t))
    with pytest.raises(ValueError, match=match):
        torch.func.grad(lambda y: ops.target_probs(y).sum())(x)
    with pytest.raises(ValueError, match=match):
        torch.func.jvp(ops.target_probs, (x,), (x,))
    for kw in (dict(temperature=t.clone().requires_grad_()),
               dict(top_p=t.clone().requires_grad_())):
        with pytest.raises(ValueError, match=match):
            ops.target_probs(x, **kw)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            ops.target_probs(x, **kw)
    with torch.inference_mode(), pytest.raises(ValueError, match="CUDA"):
        ops.target_probs(x)
    # the verified tokens are whole numbers, without a derivative
    logits, draft, u = _args()
    with pytest.raises(ValueError, match="CUDA"):
        ops.verify_sampled(logits.requires_grad_(), draft, u)


def test_misaligned_rows_at_the_c_abi():
    """Rows that do not start on their type's boundary are refused (a 16- or
    32-bit load there would fault)."""
    L = _lib.lib()
    s = _lib.Sampling(temperature_all=1.0, top_p_all=1.0)
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        for off in range(1, size):
            r = _lib.Rows(data=4096 + off, dtype=dtype, batch=2, positions=3,
                          vocab=9, stride_b=27, stride_j=9)
            p = _lib.Rows(data=4096 + off, dtype=dtype, batch=2, positions=3,
                          vocab=9, stride_b=9, row_start=4096, n_rows=6)
            for rows in (r, p):
                assert L.sg_verify_greedy(ctypes.byref(rows), 4096, None,
                                          4096, 4096, 4096, 0, None) == 1
                assert L.sg_verify_sampled(
                    ctypes.byref(rows), ctypes.byref(s), 4096, None, 4096,
                    4096, 4096, 4096, 0, None) == 1
            # without an output: 1 from the check, were it to pass as well
            assert L.sg_target_probs(ctypes.byref(r), ctypes.byref(s), None,
                                     None) == 1
    good = _lib.Rows(data=4096, dtype=0, batch=2, positions=3, vocab=9,
                     stride_b=27, stride_j=9)
    bad = _lib.Rows(data=4097, dtype=0, batch=2, positions=2, vocab=9,
                    stride_b=27, stride_j=9)
    assert L.sg_verify_probs(ctypes.byref(good), ctypes.byref(bad), 4096,
                             None, 4096, 4096, 4096, None) == 1
    # a start on the boundary passes the check (and lacks a workspace)
    assert L.sg_verify_greedy(ctypes.byref(good), 4096, None, 4096, 4096,
                              4096, 0, None) == 2


def test_refused_row_starts_and_clamps():
    draft = torch.zeros(2, 1, dtype=torch.int64)
    rows = torch.zeros(4, 5)
    for start in (torch.tensor(0), torch.zeros(3, dtype=torch.int64),
                  torch.zeros(2, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match=r"row_start must be a \[B\]"):
            ops.verify_greedy(rows, draft, row_start=start)
    L = _lib.lib()
    one = 4096  # never dereferenced
    assert L.sg_clamp_i32(None, 0, 3, 3, 1, None, None) == 0
    assert L.sg_clamp_i32(None, 3, 0, 3, 1, None, None) == 0
    assert L.sg_clamp_i32(None, 2, 3, 3, 1, one, None) == 1
    assert L.sg_clamp_i32(one, 2, 3, 3, 1, None, None) == 1
    for bad in ((-1, 3, 3, 1), (2, -1, 3, 1), (2, 3, -3, 1), (2, 3, 3, -1)):
        assert L.sg_clamp_i32(one, *bad, one, None) == 1
    assert L.sg_clamp_i32(one, 2 ** 62, 4, 4, 1, one, None) == 4
