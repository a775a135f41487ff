"""The router's balance loss, counts and gradient against the formulas in 64
bits, and the gradient against differences of the loss."""
import numpy as np
import pytest

from fp8_util import BF16, F16, F32
from gpu_util import ptr, stream

pytestmark = pytest.mark.gpu

TORCH = {F16: "float16", BF16: "bfloat16", F32: "float32"}


def reference(z, idx, mask, seq, alpha, scale):
    """(counts, prob, loss, grad) in 64 bits; z f64 [T, E]."""
    T, E = z.shape
    k, S = idx.shape[1], len(seq) - 1
    with np.errstate(invalid="ignore"):
        m = z.max(1, keepdims=True, initial=-np.inf)
        p = np.exp(z - np.where(np.isneginf(m), 0.0, m))
        tot = p.sum(1, keepdims=True)
        p = np.where(tot > 0, p / np.where(tot > 0, tot, 1.0), np.where(np.isnan(tot), np.nan, 0.0))
    counts, prob, grad = np.zeros((S, E), np.int64), np.zeros((S, E)), np.zeros((T, E))
    live = [np.arange(seq[s], seq[s + 1])[mask[seq[s]:seq[s + 1]] != 0] for s in range(S)]
    used = max(1, sum(len(t) > 0 for t in live))
    loss = 0.0
    for s, t in enumerate(live):
        if not len(t):
            continue
        r = idx[t].ravel()
        counts[s] = np.bincount(r[(r >= 0) & (r < E)], minlength=E)
        f = E * counts[s] / (k * len(t))
        prob[s] = p[t].mean(0)
        loss += alpha / used * (f * prob[s]).sum()
        grad[t] = scale * alpha / (used * len(t)) * p[t] * (f - (p[t] @ f)[:, None])
    return counts, prob, loss, grad


def balance(L, z, code, idx, mask, seq, alpha=0.01, scale=1.0, ldl=None, grad=True, st=None):
    import torch
    T, E = z.shape
    dt = getattr(torch, TORCH[code])
    k, S = idx.shape[1], 1 if seq is None else len(seq) - 1
    dz = torch.full((T, ldl or E), float("nan"), dtype=dt, device="cuda")
    dz[:, :E] = torch.from_numpy(z).cuda().to(dt)
    zv = dz[:, :E].double().cpu().numpy()
    di = torch.from_numpy(np.ascontiguousarray(idx, np.int32)).cuda()
    dm = None if mask is None else torch.from_numpy(mask.astype(np.uint8)).cuda()
    ds = None if seq is None else torch.from_numpy(np.asarray(seq, np.int32)).cuda()
    counts = torch.full((S, E), -1, dtype=torch.int32, device="cuda")
    prob, loss = torch.full((S, E), -1.0, device="cuda"), torch.full((1,), -1.0, device="cuda")
    g = torch.full((T, (ldl or E) + 1), -7.0, dtype=dt, device="cuda")
    n = L.ts_cuda_router_balance_work(S, E)
    work = torch.full((n + 8,), 0xA5, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    rc = L.ts_cuda_op_router_balance(ptr(dz), code, dz.stride(0), ptr(di), None if dm is None else ptr(dm),
                                     None if ds is None else ptr(ds), S, T, E, k, alpha, scale, ptr(counts), ptr(prob),
                                     ptr(loss), ptr(g) if grad else None, g.stride(0), ptr(work), n,
                                     stream() if st is None else st)
    assert rc == 0, L.ts_cuda_last_error()
    torch.cuda.synchronize()
    assert (work[n:] == 0xA5).all()
    assert (g[:, E:].float() == -7.0).all()
    if not grad:
        assert (g.float() == -7.0).all()
    return (counts.cpu().numpy(), prob.cpu().numpy(), float(loss[0]), g[:, :E].double().cpu().numpy()), zv


def make(rng, T, E, k, S):
    z = (rng.standard_normal((T, E)) * 1.5 + rng.standard_normal(E) * 0.7).astype(np.float32)
    idx = np.argsort(-z, 1, kind="stable")[:, :k].astype(np.int32)
    cuts = np.sort(rng.integers(0, T + 1, S - 1))  # empty documents among them
    return z, idx, (rng.random(T) < 0.9).astype(np.uint8), np.concatenate([[0], cuts, [T]])


def compare(got, ref, code, E, T):
    """Counts exact; prob and loss: a softmax in f32 (its exponential, sum of E terms and division) is off by at most
    (E + 8) 2^-24 relative, a sum over tokens in pieces of any order by (T + 2) 2^-24 at the very most; grad: p (f - mean)
    with the same errors in p, in the mean and in the f32 factors, then rounded to its type."""
    eps = 2.0 ** -24
    assert np.array_equal(got[0], ref[0])
    rel = (E + 16 + min(T, 1024)) * eps
    assert np.allclose(got[1], ref[1], rtol=rel, atol=2.0 ** -40)
    assert abs(got[2] - ref[2]) <= (rel + 4 * eps) * abs(ref[2]) + 1e-30
    half = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: eps}[code]
    tiny = 2.0 ** -25 if code == F16 else 1e-38
    # |p (f - mean)| <= p f + p mean: the terms cancel, so the bound goes by their sizes
    size = ref[4]
    off = np.abs(got[3] - ref[3])
    bound = (2 * E + 32) * eps * size + half * np.abs(ref[3]) + tiny
    assert (off <= bound).all(), (off - bound).max()


def term_sizes(z, idx, mask, seq, alpha, scale):
    """Upper sizes of the two terms of each gradient element."""
    counts, prob, loss, grad = reference(z, idx, mask, seq, alpha, scale)
    T, E = z.shape
    size = np.zeros((T, E))
    used = max(1, sum(bool(mask[seq[s]:seq[s + 1]].any()) for s in range(len(seq) - 1)))
    for s in range(len(seq) - 1):
        t = np.arange(seq[s], seq[s + 1])[mask[seq[s]:seq[s + 1]] != 0]
        if len(t):
            f = E * counts[s] / (idx.shape[1] * len(t))
            p = np.exp(z[t] - z[t].max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            size[t] = scale * alpha / (used * len(t)) * p * (f + (p @ f)[:, None])
    return counts, prob, loss, grad, size


@pytest.mark.parametrize("code", [F16, BF16, F32])
@pytest.mark.parametrize("T,E,k,S", [(1, 2, 1, 1), (1, 128, 4, 1), (7, 128, 4, 1), (80, 128, 4, 1), (33, 31, 2, 3),
                                     (500, 1, 1, 2), (1000, 60, 6, 17), (2049, 128, 4, 5), (300, 257, 8, 300),
                                     (129, 1024, 64, 2), (4097, 256, 8, 40), (9001, 33, 3, 2)])
def test_balance(cuda_lib, T, E, k, S, code):
    rng = np.random.default_rng(T * 13 + E)
    z, idx, mask, seq = make(rng, T, E, k, S)
    scale = 4096.0 if code == F16 else 1.0
    got, zv = balance(cuda_lib, z, code, idx, mask, seq, scale=scale, ldl=E + T % 4)
    compare(got, term_sizes(zv, idx, mask, seq, 0.01, scale), code, E, T)


@pytest.mark.parametrize("T,E", [(77, 128), (3000, 24)])
def test_balance_without_mask_sequences_or_gradient(cuda_lib, T, E):
    rng = np.random.default_rng(T)
    z, idx, _, _ = make(rng, T, E, 2, 1)
    one = np.ones(T, np.uint8)
    got, zv = balance(cuda_lib, z, F32, idx, None, None)
    compare(got, term_sizes(zv, idx, one, [0, T], 0.01, 1.0), F32, E, T)
    bare, _ = balance(cuda_lib, z, F32, idx, None, None, grad=False)
    assert np.array_equal(bare[0], got[0]) and np.array_equal(bare[1], got[1]) and bare[2] == got[2]


def test_balance_gradient_against_differences(cuda_lib):
    """Central differences of the 64-bit loss with the counts held: the operator's gradient along random directions."""
    rng = np.random.default_rng(4)
    T, E, k, S = 60, 40, 4, 3
    z, idx, mask, seq = make(rng, T, E, k, S)
    got, zv = balance(cuda_lib, z, F32, idx, mask, seq, alpha=1.0)
    h = 1e-4
    for _ in range(5):
        d = rng.standard_normal((T, E))
        hi, lo = (reference(zv + s * h * d, idx, mask, seq, 1.0, 1.0)[2] for s in (1, -1))
        slope = (hi - lo) / (2 * h)
        size = term_sizes(zv, idx, mask, seq, 1.0, 1.0)[4]
        # the third derivative's h^2 / 6 and the rounding of the 64-bit losses over 2 h
        far = (2 * E + 32) * 2.0 ** -24 * (size * np.abs(d)).sum() + h * h * (size * np.abs(d) ** 3).sum() * 8 + 1e-16 / h * 10
        assert abs((got[3] * d).sum() - slope) <= far


def test_balance_masked_experts_and_rows(cuda_lib):
    """-inf closes experts to a token, and a row with none open has no probability and no gradient."""
    rng = np.random.default_rng(9)
    T, E, k = 300, 128, 4
    z, idx, mask, seq = make(rng, T, E, k, 2)
    z[rng.random((T, E)) < 0.3] = -np.inf
    z[5] = -np.inf
    z[6, 1:] = -np.inf
    mask[5:7] = 1
    got, zv = balance(cuda_lib, z, F32, idx, mask, seq)
    ref = reference(zv, idx, mask, seq, 0.01, 1.0)
    assert np.array_equal(got[0], ref[0])
    assert np.allclose(got[1], ref[1], rtol=600 * 2.0 ** -24, atol=2.0 ** -40)
    assert abs(got[2] - ref[2]) <= 1e-4 * abs(ref[2])
    assert (got[3][5] == 0).all() and (got[3][np.isneginf(zv)] == 0).all()
    assert np.isfinite(got[3]).all()
    low = z.copy()
    low[np.isneginf(low)] = np.finfo(np.float32).min  # the lowest value closes them just as well, but for the empty row
    low[5] = z[5]
    same, _ = balance(cuda_lib, low, F32, idx, mask, seq)
    for a, b in zip(got, same):
        assert np.array_equal(a, b)


def test_balance_nan_stays_in_its_document(cuda_lib):
    rng = np.random.default_rng(10)
    T, E, k = 90, 64, 2
    z, idx, mask, _ = make(rng, T, E, k, 1)
    seq = np.array([0, 30, 60, 90])
    mask[:] = 1
    mask[70] = 0
    z[40, 3], z[41, 5], z[70] = np.nan, np.inf, np.nan
    got, _ = balance(cuda_lib, z, F32, idx, mask, seq)
    assert np.isnan(got[1][1]).all() and np.isfinite(got[1][[0, 2]]).all() and np.isnan(got[2])
    assert np.isnan(got[3][40:42]).all()
    rest = np.delete(got[3], [40, 41], 0)
    assert np.isfinite(rest).all() and (got[3][70] == 0).all()


def test_balance_dropped_routes_and_tokens_outside(cuda_lib):
    rng = np.random.default_rng(12)
    T, E, k = 200, 16, 4
    z, idx, mask, _ = make(rng, T, E, k, 1)
    idx[rng.random((T, k)) < 0.2] = -1
    idx[3, 0], idx[4, 1] = E, 1 << 30
    got, zv = balance(cuda_lib, z, F32, idx, mask, [20, 90, 90, 150])
    inside = mask.copy()
    inside[:20], inside[150:] = 0, 0
    compare(got, term_sizes(zv, idx, inside, [0, 90, 90, 200], 0.01, 1.0), F32, E, T)
    assert (got[3][:20] == 0).all() and (got[3][150:] == 0).all()


def test_balance_of_no_tokens(cuda_lib):
    """Every token masked, or none at all: zeros, not NaN."""
    z, idx = np.zeros((40, 8), np.float32), np.zeros((40, 2), np.int32)
    got, _ = balance(cuda_lib, z, F32, idx, np.zeros(40, np.uint8), [0, 10, 40])
    assert not got[0].any() and not got[1].any() and got[2] == 0 and not got[3].any()
    got, _ = balance(cuda_lib, z[:0], F32, idx[:0], None, None)
    assert not got[0].any() and not got[1].any() and got[2] == 0


def test_balance_repeats_bit_for_bit(cuda_lib):
    import torch
    rng = np.random.default_rng(13)
    z, idx, mask, seq = make(rng, 20000, 128, 4, 9)
    s = torch.cuda.Stream()
    first, _ = balance(cuda_lib, z, F32, idx, mask, seq)
    for st in (None, s.cuda_stream, None):
        again, _ = balance(cuda_lib, z, F32, idx, mask, seq, st=st)
        for a, b in zip(first, again):
            assert np.array_equal(a, b)


def test_balance_of_equal_counts(cuda_lib):
    """Every expert takes every token: nothing to balance, a gradient of exactly zero and a loss of alpha."""
    rng = np.random.default_rng(14)
    for T, E in ((50, 4), (3000, 8)):
        z = rng.standard_normal((T, E)).astype(np.float32) * 3
        idx = np.tile(np.arange(E, dtype=np.int32), (T, 1))
        got, _ = balance(cuda_lib, z, F32, idx, None, None, alpha=0.5)
        assert (got[0] == T).all() and not got[3].any()
        assert abs(got[2] - 0.5) <= 0.5 * (E + 16 + min(T, 1024)) * 2.0 ** -24
