"""Attention over the 4-bit KV cache where its values' scales are small, large or
both, against 64-bit results over the values that the cache holds: the size of V
costs no accuracy, and neither does a key that a row does not see or hardly weighs.

Bounds (e = 2^-24, half an f32 step), all relative to what a row sees: scores,
exponentials, sums and pieces as in the other tests of this cache, 2 e ((terms +
16) S + n + 64) of sum p |v|.  Beside that a weight enters in two f16 pieces, whose
second rounds at 2^-25 at the finest while the largest weight is 2^10 or more:
  values in two pieces (many rows): 2^-35 |v| of each key, scales below 32;
  weights times scales (fewer rows), scales in [2^-11, 2): 2^-35 |code| <= e |v|;
  weights times scales, raised so that the largest of 32 keys is 2^14 or more: 2^-39 of
  that largest product times a code of up to 8, n 2^-36 max p D;
each over the normaliser in units of the largest weight."""
import numpy as np
import pytest

import vlrf_amd as V
from vlrf_amd import formats as F

pytestmark = pytest.mark.gpu

# (H, G, d, T): a column a row and block; 16 rows a workgroup of eight and of four waves; many rows.
FEW = [(8, 2, 64, 1), (32, 8, 128, 1), (8, 2, 128, 3)]
BLOCKS = [(32, 8, 128, 33), (64, 8, 64, 40), (128, 8, 128, 40), (256, 16, 64, 40)]
TILES = [(128, 128, 64, 300), (256, 64, 128, 150)]


def _stored(x, G, d):
    """The values [n, G, d] and block scales, as wide, that the cache holds of rows x."""
    x = np.ascontiguousarray(x, np.float32)
    blocks = F.quantize(x, V.DT_Q4_0)
    scale = np.abs(blocks.reshape(-1, 18)[:, :2].copy().view(np.float16).astype(np.float64)).ravel()
    return F.dequantize(blocks, V.DT_Q4_0, x.size).reshape(-1, G, d), scale.repeat(32).reshape(-1, G, d)


def _check(got, q, K, Vv, D, H, scale, terms, many):
    """got, q [T, H, d]; K, Vv, D [n, G, d]: values and V's scales; many: the values may stand in two pieces."""
    T, _, d = q.shape
    n, G, _ = K.shape
    q, K, Vv = (t.astype(np.float64) for t in (q, K, Vv))
    keep = np.arange(n)[None, :] <= np.arange(T)[:, None] + (n - T)
    worst = 0.0
    for h in range(H):
        k, v, s = K[:, h // (H // G)], Vv[:, h // (H // G)], D[:, h // (H // G)]
        x = np.where(keep, q[:, h] @ k.T * float(scale), -np.inf)
        p = np.exp(x - x.max(1, keepdims=True))
        L = p.sum(1, keepdims=True)
        S = np.where(keep, np.abs(q[:, h]) @ np.abs(k).T * abs(float(scale)), 0).max(1, keepdims=True)
        floor = 2.0 ** -24 * keep @ (np.abs(v) * ((s >= 2.0 ** -11) & (s < 2)))
        if many:
            floor += 2.0 ** -35 * keep @ (np.abs(v) * (s < 32))
        floor += n * 2.0 ** -36 * np.stack([(p[t][:, None] * s).max(0) for t in range(T)])
        bound = (2 * 2.0 ** -24 * ((terms + 16) * S + n + 64) * (p @ np.abs(v)) + floor) / L
        ratio = np.abs(got[:, h] - p @ v / L) / bound
        assert np.isfinite(got[:, h]).all()
        worst = max(worst, ratio.max())
    print(f"  largest error / bound {worst:.3g}", flush=True)
    assert worst <= 1


def _queries(T, H, d, seed, size=1.0):
    """Queries with one element that is not zero, so that scores cost few roundings."""
    q = np.zeros((T * H, d), np.float32)
    at = np.arange(T * H)
    q[at, at * 7 % d] = F.normal(seed, "q", T * H, size)
    return q.reshape(T, H, d)


def _run(ctx, K, Vv, n, q, G, scale, cap=None):
    """Rows K, Vv appended and all from n on forgotten again; the attention of q over the rest."""
    T, H, d = q.shape
    kv = V.KVCache(ctx, 1, cap or len(K), G, d, V.KV_Q4_0)
    kv.append(0, ctx.to_device(K), ctx.to_device(Vv), len(K))
    kv.truncate(0, n)
    out = ctx.alloc(q.nbytes)
    kv.attention_chunk(0, ctx.to_device(q), out, H, T, n, scale)
    return out.download(q.shape)


@pytest.mark.parametrize("H,G,d,T", FEW + BLOCKS + TILES)
@pytest.mark.parametrize("v_std", [1e-2, 1e-3, 1e-4, 1e-5, 1e-6])
def test_small_values(ctx, v_std, H, G, d, T):
    """Values of any size down to f16's smallest scales."""
    print(f"[case] kv4 small values v={v_std} H={H} G={G} d={d} T={T}", flush=True)
    n = max(T, 70)
    K, Vv = F.normal(110, "k", n * G * d).reshape(n, -1), F.normal(110, "v", n * G * d, v_std).reshape(n, -1)
    q = _queries(T, H, d, 110)
    got = _run(ctx, K, Vv, n, q, G, 0.5)
    _check(got, q, _stored(K, G, d)[0], *_stored(Vv, G, d), H, 0.5, 1, T > 100)


@pytest.mark.parametrize("H,G,d,T", FEW + BLOCKS + TILES)
@pytest.mark.parametrize("v_std", [5e-7, 2e-7])
def test_smallest_values(ctx, v_std, H, G, d, T):
    """Values whose scales are a few of f16's smallest steps, few keys."""
    print(f"[case] kv4 smallest values v={v_std} H={H} G={G} d={d} T={T}", flush=True)
    n = max(T, 40)
    K, Vv = F.normal(116, "k", n * G * d).reshape(n, -1), F.normal(116, "v", n * G * d, v_std).reshape(n, -1)
    q = _queries(T, H, d, 116)
    got = _run(ctx, K, Vv, n, q, G, 0.5)
    _check(got, q, _stored(K, G, d)[0], *_stored(Vv, G, d), H, 0.5, 1, T > 100)


@pytest.mark.parametrize("H,G,d,T", FEW + BLOCKS + TILES)
@pytest.mark.parametrize("large", [30.0, 1e4, 1e5])
def test_forgotten_large_values(ctx, large, H, G, d, T):
    """Finite large rows behind the context, left there by a truncation, beside small and usual values."""
    print(f"[case] kv4 forgotten v={large} H={H} G={G} d={d} T={T}", flush=True)
    n = max(T, 70) + 7
    more = 40
    K, Vv = F.normal(111, "k", (n + more) * G * d).reshape(n + more, -1), F.normal(111, "v", (n + more) * G * d).reshape(n + more, -1)
    Vv[:n, :32] *= 1e-3
    Vv[n - 3:n] *= 0.01
    Vv[n:] *= large
    q = _queries(T, H, d, 111)
    got = _run(ctx, K, Vv, n, q, G, 0.5)
    _check(got, q, _stored(K[:n], G, d)[0], *_stored(Vv[:n], G, d), H, 0.5, 1, T > 100)


@pytest.mark.parametrize("H,G,d,T", [s for s in FEW + BLOCKS + TILES if s[3] > 1])
@pytest.mark.parametrize("large", [30.0, 1e4, 1e5])
def test_hidden_large_values(ctx, large, H, G, d, T):
    """Finite large rows that a chunk's later rows see and its earlier ones do not."""
    print(f"[case] kv4 hidden v={large} H={H} G={G} d={d} T={T}", flush=True)
    n = max(T, 70)
    K, Vv = F.normal(112, "k", n * G * d).reshape(n, -1), F.normal(112, "v", n * G * d, 1e-3).reshape(n, -1)
    Vv[n - T + 1::5] *= 1e3 * large
    q = _queries(T, H, d, 112)
    got = _run(ctx, K, Vv, n, q, G, 0.5)
    K, (Vv, D) = _stored(K, G, d)[0], _stored(Vv, G, d)
    _check(got, q, K, Vv, D, H, 0.5, 1, T > 100)
    _check(got[:1], q[:1], K[:n - T + 1], Vv[:n - T + 1], D[:n - T + 1], H, 0.5, 1, T > 100)   # the row that sees none of them


@pytest.mark.parametrize("H,G,d,T", FEW + BLOCKS + TILES)
@pytest.mark.parametrize("weight", [10.0, 16.0, 24.0])
def test_large_values_of_small_weight(ctx, weight, H, G, d, T):
    """Values near f16's largest scale whose keys weigh e^-weight of the others, beside values of 1e-3."""
    print(f"[case] kv4 large values that weigh e^-{weight} H={H} G={G} d={d} T={T}", flush=True)
    n = max(T, 70)
    K, Vv = F.normal(113, "k", n * G * d, 0.01).reshape(n, G, d), F.normal(113, "v", n * G * d, 1e-3).reshape(n, -1)
    big = np.arange(n) % 6 == 3
    K[big, :, 0], K[~big, :, 0] = -1.0, 1.0
    Vv[big] *= 8e7
    q = np.zeros((T, H, d), np.float32)
    q[..., 0] = weight * (1 + 0.01 * F.normal(113, "q", T * H).reshape(T, H))
    got = _run(ctx, K.reshape(n, -1), Vv, n, q, G, 0.5)
    _check(got, q, _stored(K.reshape(n, -1), G, d)[0], *_stored(Vv, G, d), H, 0.5, 1, T > 100)


@pytest.mark.parametrize("H,G,d,T", FEW + BLOCKS)
def test_scales_at_the_borders(ctx, H, G, d, T):
    """Scales on and next to 2^-11 and 2, zero, f16's smallest, its largest, and none that a row weighs alike."""
    print(f"[case] kv4 borders H={H} G={G} d={d} T={T}", flush=True)
    n = 97
    K, Vv = F.normal(114, "k", n * G * d).reshape(n, -1), np.empty((n, G * d), np.float32)
    step = 2.0 ** -10
    scales = [2.0 ** -11, 2.0 ** -11 * (1 - step / 2), 2.0 ** -11 * (1 + step), 2.0, 2 * (1 - step / 2), 2 * (1 + step), 0.0, 2.0 ** -24,
              3 * 2.0 ** -24, 2.0 ** -14, 65504.0, 1.0, 0.25]
    codes = np.rint(F.normal(114, "c", n * G * d, 3.0)).clip(-7, 7).reshape(n, G * d // 32, 32)
    codes[:, :, 5] = -8
    for j in range(n):
        for b in range(G * d // 32):
            Vv[j, 32 * b:32 * b + 32] = codes[j, b] * scales[(j * 5 + b + j // 32) % len(scales)]
    q = _queries(T, H, d, 114)
    got = _run(ctx, K, Vv, n, q, G, 0.5)
    _check(got, q, _stored(K, G, d)[0], *_stored(Vv, G, d), H, 0.5, 1, False)


@pytest.mark.parametrize("H,G,d", [(32, 8, 128), (32, 4, 64)])
def test_small_and_large_values_behind_many_keys(ctx, H, G, d):
    """Several groups of keys a wave, of which some have small scales, some large ones and most neither."""
    print(f"[case] kv4 mixed groups H={H} G={G} d={d}", flush=True)
    n = 6001
    K, Vv = F.normal(115, "k", n * G * d).reshape(n, -1), F.normal(115, "v", n * G * d).reshape(n, -1)
    Vv[1000:1500] *= 1e-5
    Vv[1234] *= 1e6
    Vv[3000::711] *= 1e4
    Vv[5000:5003] = 0
    for T in (1, 5):
        q = _queries(T, H, d, 115, 4.0)
        got = _run(ctx, K, Vv, n, q, G, 0.5)
        _check(got, q, _stored(K, G, d)[0], *_stored(Vv, G, d), H, 0.5, 1, False)
