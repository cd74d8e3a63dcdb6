"""4-bit KV cache on the GPU at the ends of its ranges: padding rows whatever the norm, weights and values
far below the largest, scores past the range in which fp32 holds fractions, scales that are not finite.
The documented errors of the attention are those of fp32 arithmetic, with few rows for a weight times its
V scale down to 2^-50 of the row's largest weight times the largest scale read."""
import numpy as np
import pytest

import kv_q4_ref as R
import vsl
from test_kv_q4_gpu import Cache, dev, rope_tables, status_word

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kvdt", [vsl.Q4_0, vsl.F16, vsl.F32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("style", [vsl.ROPE_ADJACENT, vsl.ROPE_HALVES])
@pytest.mark.parametrize("n", [6, 3000])
def test_padding_rows_are_zero_whatever_the_norm(kvdt, hd, style, n):
    """eps 0, and norm weights and rotation factors that are not finite."""
    nh, nkv, page = 8, 2, 64
    c = Cache(kvdt, 4, nkv, hd, page, [[0, 1], [2, -1]])
    before = c.k.clone(), c.v.clone()
    x = torch.randn(n, (nh + 2 * nkv) * hd, device="cuda")
    w = torch.ones(hd, device="cuda")
    w[3] = float("inf")
    cos, sin = (dev(a) for a in rope_tables(128, hd))
    cos[0, 1] = float("nan")
    seq = torch.arange(n, device="cuda", dtype=torch.int32) % 3
    pad = torch.full_like(seq, -1)
    for norms in ((w, w), (w, None), (torch.ones_like(w), torch.ones_like(w))):
        c.status.zero_()
        q = c.append(x, nh, *norms, seq, pad, cos, sin, style, eps=0.0)
        assert (q == 0).all() and c.status.item() == 0
        q = c.append(x, nh, *norms, seq, pad + 129, cos, sin, style, eps=0.0)  # past the table
        assert (q == 0).all() and c.status.item() == -5
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])


def values(codes, sc):
    """codes [2, pages, nkv, page, hd], scales [2, pages, nkv, page, hd / 32] -> K, V float64 [nkv, len, hd]."""
    with np.errstate(invalid="ignore"):
        x = (codes.astype(np.float64) - 8) * np.repeat(sc.astype(np.float64), 32, -1)
    return x.transpose(0, 2, 1, 3, 4).reshape(2, codes.shape[2], -1, codes.shape[-1])


def attend(q, codes, sc, pos, mask=None):
    """q fp32 [rows, nh, hd] of one sequence whose pages are codes, sc in order; status has to stay 0."""
    (rows, nh, hd), (_, pages, nkv, page, _) = q.shape, codes.shape
    kc, vc = (dev(R.pack(codes[i], sc[i], page, bool(i))) for i in range(2))
    out, st = torch.full((rows, nh, hd), 7.0, device="cuda"), status_word()
    n = vsl.flash_decode_q4_workspace_size(1, rows, nh, nkv, hd)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    vsl.flash_decode_q4(dev(q), kc, vc, pages, dev(np.arange(pages, dtype=np.int32)[None]), pages, page,
                        dev(np.array([pos], np.int32)), 1, rows, nh, nkv, hd, out, ws, n, sparse=mask, status=st)
    assert st.item() == 0
    return out.cpu().numpy().astype(np.float64)


def floor_of(q, codes, sc, pos):
    """What the documented limit of 2^-50 adds to an element's error: [rows, nh, hd]."""
    k, _ = values(codes, sc)
    rows, nh, hd = q.shape
    nkv = k.shape[0]
    out = np.zeros((rows, nh, hd))
    for r in range(rows):
        n = pos + r + 1
        for h in range(nh):
            g = h * nkv // nh
            s = k[g, :n] @ q[r, h].astype(np.float64) / np.sqrt(hd)
            w = np.exp(s - s.max())
            top = np.abs(sc[1].astype(np.float64)[:, g]).max()
            c = np.abs(codes[1][:, g].reshape(-1, hd)[:n].astype(np.float64) - 8).sum(0)
            out[r, h] = 2.0 ** -50 * (w / w.sum()).max() * top * c
    return out


def random_cache(rng, pages, nkv, hd, k_scale=0.2, v_scale=0.2, page=64):
    codes = rng.integers(0, 16, (2, pages, nkv, page, hd)).astype(np.uint8)
    sc = rng.standard_normal((2, pages, nkv, page, hd // 32))
    sc[0] *= k_scale
    sc[1] *= v_scale
    return codes, sc.astype(np.float16)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (8, 2), (8, 1)])
@pytest.mark.parametrize("k", [24, 28, 36, 42])
def test_weights_far_below_the_largest(hd, nh, nkv, k):
    """The first position has all the weight and the value 0: the output is what the others, of weights
    around 2^-k, add up to."""
    rng = np.random.default_rng(hd + nh + nkv + k)
    codes, sc = random_cache(rng, 5, nkv, hd, k_scale=0.01)
    codes[0, 0, :, 0], sc[0, 0, :, 0] = 15, np.float16(k * np.log(2) / (7 * np.sqrt(hd)))
    codes[1, 0, :, 0] = 8
    q = (1 + 0.1 * rng.standard_normal((1, nh, hd))).astype(np.float32)
    got = attend(q, codes, sc, 299)
    kk, vv = values(codes, sc)
    want, tol = R.attention(q.astype(np.float64), kk[:, :300], vv[:, :300], 299)
    tol += floor_of(q, codes, sc, 299)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (8, 2), (8, 1)])
@pytest.mark.parametrize("r", [20, 30])
def test_a_block_of_much_larger_values(hd, nh, nkv, r):
    """One block's V scales are 2^r times another's."""
    rng = np.random.default_rng(hd + nh + nkv + r)
    codes, sc = random_cache(rng, 5, nkv, hd, v_scale=2.0 ** -15)
    sc[1, ..., 0] = (rng.standard_normal(sc[1, ..., 0].shape) * 2.0 ** (r - 17)).astype(np.float16)
    q = rng.standard_normal((1, nh, hd)).astype(np.float32)
    got = attend(q, codes, sc, 299)
    kk, vv = values(codes, sc)
    want, tol = R.attention(q.astype(np.float64), kk[:, :300], vv[:, :300], 299)
    tol += floor_of(q, codes, sc, 299)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,rows", [(2, 1), (8, 1), (4, 4)])
@pytest.mark.parametrize("scale", [0x7bff, 0x3bff])
def test_large_scores_with_full_mantissas(hd, nh, rows, scale):
    """Scores of 1e4 and more, V scales with every bit of the mantissa set: finite, and inside the bounds."""
    for seed in range(6):
        rng = np.random.default_rng(100 * hd + 10 * nh + seed)
        codes, sc = random_cache(rng, 3, 1, hd)
        sc[1] = np.array([scale], np.uint16).view(np.float16)[0]
        q = (rng.standard_normal((rows, nh, hd)) * 10.0 ** rng.uniform(3, 5)).astype(np.float32)
        pos = 150 - rows
        got = attend(q, codes, sc, pos)
        kk, vv = values(codes, sc)
        want, tol = R.attention(q.astype(np.float64), kk[:, :150], vv[:, :150], pos)
        assert (np.abs(got - want) <= tol).all(), seed


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,rows", [(2, 1), (8, 1), (4, 4)])
@pytest.mark.parametrize("size", [3e5, 3e7, 1.7e9, 1e12, 1e30])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(hd, nh, rows, size, sign):
    """One dimension of q counts. Its best positions are two of equal score, all others far below them:
    the output is the mean of the two values, however large the scores."""
    rng = np.random.default_rng(hd + nh + rows)
    codes, sc = random_cache(rng, 3, 1, hd)
    sc[1] = np.array([0x3bff], np.uint16).view(np.float16)[0]
    codes[0, ..., 0] = np.where(sign > 0, 2, 14)  # values of q's dimension: -6 d or 6 d, d = 1 ...
    sc[0, ..., 0] = 1.0
    a, b = 3, 77
    for t in (a, b):
        codes[0, t // 64, :, t % 64, 0] = 12  # ... but 4 d at the two
    q = np.zeros((rows, nh, hd), np.float32)
    q[..., 0] = sign * size * (1 + rng.random((rows, nh)))
    if sign < 0:  # negative scores: the two are the least negative
        codes[0, ..., 0] = np.where(codes[0, ..., 0] == 12, 9, 14)
    got = attend(q, codes, sc, 150 - rows)
    vv = values(codes, sc)[1][0]
    want = np.broadcast_to((vv[a] + vv[b]) / 2, got.shape)
    assert (np.abs(got - want) <= 2.0 ** -18 * np.abs(vv[[a, b]]).max(0)).all(), float(np.abs(got - want).max())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (8, 2), (8, 1)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n", [20, 300])
def test_a_scale_that_is_not_finite_leaves_the_other_blocks_alone(hd, nh, nkv, bad, n):
    """Small scales beside it keep their digits."""
    rng = np.random.default_rng(hd + nh + nkv)
    codes, sc = random_cache(rng, 5, nkv, hd, k_scale=0.02, v_scale=2.0 ** -21)
    codes[1, 0, :, 9, 32:64] = 8 + rng.integers(1, 8, 32)  # no code 8: times an infinity that is NaN as well
    sc[1, 0, :, 9, 1] = bad
    q = rng.standard_normal((1, nh, hd)).astype(np.float32)
    got = attend(q, codes, sc, n - 1)
    assert not np.isfinite(got[..., 32:64]).any()
    clean = sc.copy()
    clean[1, 0, :, 9, 1] = 0
    kk, vv = values(codes, clean)
    want, tol = R.attention(q.astype(np.float64), kk[:, :n], vv[:, :n], n - 1)
    tol += floor_of(q, codes, clean, n - 1)
    rest = [d for d in range(hd) if not 32 <= d < 64]
    assert (np.abs(got - want) <= tol)[..., rest].all(), float((np.abs(got - want) / tol)[..., rest].max())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,rows", [(2, 1), (8, 1), (8, 16)])
@pytest.mark.parametrize("n", [20, 150])
def test_scores_past_the_range_of_fp32_are_no_zeros(hd, nh, rows, n):
    """Finite queries whose scores overflow: NaN, as for infinite ones, and only in their head."""
    rng = np.random.default_rng(hd + nh + rows)
    codes, sc = random_cache(rng, 3, 1, hd)
    codes[0, ..., 0], sc[0, ..., 0] = 12, 8.0
    q = rng.standard_normal((rows, nh, hd)).astype(np.float32)
    fine = attend(q, codes, sc, n - rows)
    q[0, 1], q[0, 1, 0] = 0.0, 3e38
    got = attend(q, codes, sc, n - rows)
    keep = np.ones((rows, nh), bool)
    keep[0, 1] = False
    assert np.isfinite(fine).all() and np.isnan(got[0, 1]).all() and np.array_equal(got[keep], fine[keep])


# ---- rows enough for tiles of 128 columns ----

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [0x7bff, 0x3bff])
def test_chunk_large_scores_with_full_mantissas(hd, scale):
    rows, nh, pos = 16, 8, 134
    for seed in range(6):
        rng = np.random.default_rng(100 * hd + 10 * nh + seed)
        codes, sc = random_cache(rng, 3, 1, hd)
        sc[1] = np.array([scale], np.uint16).view(np.float16)[0]
        q = (rng.standard_normal((rows, nh, hd)) * 10.0 ** rng.uniform(3, 5)).astype(np.float32)
        got = attend(q, codes, sc, pos)
        kk, vv = values(codes, sc)
        want, tol = R.attention(q.astype(np.float64), kk[:, :150], vv[:, :150], pos)
        # where the heaviest positions have code 8, the documented limit of 2^-50 shows
        assert (np.abs(got - want) <= tol + floor_of(q, codes, sc, pos)).all(), seed


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [3e5, 3e7, 1.7e9, 1e12, 1e30])
@pytest.mark.parametrize("sign", [1, -1])
def test_chunk_scores_of_any_size(hd, size, sign):
    test_scores_of_any_size(hd, 8, 16, size, sign)
