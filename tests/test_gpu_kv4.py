"""The 4-bit KV cache on the GPU: appends bit for bit as the host encoder's
blocks, the rows read back, and attention of one token and of chunks of tokens
against 64-bit results over the values that the cache holds.

Bounds on attention (e = 2^-24, half an f32 step): a score sums d products of q
in two f16 pieces (2^-21 each at most, 8 e) and exact codes, scaled by block: (d
+ 16) e S, S the row's largest |scale| sum |q||k|.  A weight adds the exponential
and its own two pieces (64 e together), the sums over n keys n e, each in the
numerator and in the normaliser.  The second piece of a weight times a block's
scale rounds at 2^-34 at the finest, against codes of up to 8: n 2^-31 over the
normaliser."""
import ctypes as C

import numpy as np
import pytest

import vlrf_amd as V
from vlrf_amd import _lib
from vlrf_amd import formats as F

pytestmark = pytest.mark.gpu


def _attention64(q, K, Vv, n_heads, scale, terms=None):
    """(result [T, H, d], bound) for q [T, H, d] and the cache's values K, Vv [n, G, d]; terms: the
    products that a score adds up where they are fewer than d."""
    T, _, d = q.shape
    terms = terms or d
    n, G, _ = K.shape
    q, K, Vv = (t.astype(np.float64) for t in (q, K, Vv))
    keep = np.arange(n)[None, :] <= np.arange(T)[:, None] + (n - T)
    out, bound = np.empty((T, n_heads, d)), np.empty((T, n_heads, d))
    for h in range(n_heads):
        k, v = K[:, h // (n_heads // G)], Vv[:, h // (n_heads // G)]
        s = np.where(keep, q[:, h] @ k.T * scale, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        L = p.sum(1, keepdims=True)
        p /= L
        S = np.where(keep, np.abs(q[:, h]) @ np.abs(k).T * abs(scale), 0).max(1, keepdims=True)
        out[:, h] = p @ v
        bound[:, h] = 2 * 2.0 ** -24 * ((terms + 16) * S + n + 64) * (p @ np.abs(v)) + n * 2.0 ** -31 / L
    return out, bound


def _filled(ctx, n, G, d, seed, more=0, k_std=1.0, v_std=1.0, layers=1):
    """A cache with n + more rows in its last layer, and their values."""
    row = G * d
    K = F.normal(seed, "kv4.k", (n + more) * row, k_std).reshape(-1, row)
    Vv = F.normal(seed, "kv4.v", (n + more) * row, v_std).reshape(-1, row)
    kv = V.KVCache(ctx, layers, n + more, G, d, V.KV_Q4_0)
    kv.append(layers - 1, ctx.to_device(K), ctx.to_device(Vv), n + more)
    return kv, _decoded(K, n, G, d), _decoded(Vv, n, G, d)


def _decoded(x, n, G, d):
    x = np.ascontiguousarray(x[:n])
    return F.dequantize(F.quantize(x, V.DT_Q4_0), V.DT_Q4_0, x.size).reshape(n, G, d)


def _special_rows(row):
    x = F.normal(81, "kv4.special", 8 * row).reshape(8, row)
    x[0] = 0
    x[1, ::2], x[1, 1::2] = 0.75, -0.75                 # equal magnitudes: the first one's sign decides
    x[2, ::2], x[2, 1::2] = -0.75, 0.75
    x[3] *= 1e-7                                        # scales below f16's normal range
    x[4] *= 1e-9                                        # scales of zero
    x[5] *= 1e5                                         # scales near f16's largest
    x[6, :16] = np.linspace(-8.5, 8.5, 16)              # codes on and next to the border
    x[7] = np.round(x[7] * 2) / 2                       # ties between codes
    return x.astype(np.float32)


@pytest.mark.parametrize("G,d,T,base", [(1, 64, 1, 0), (4, 64, 333, 0), (8, 128, 9, 5), (2, 96, 70, 31), (3, 32, 40, 100),
                                        (1, 256, 33, 7), (5, 64, 1, 63), (8, 128, 257, 64)])
def test_append_is_the_host_encoder(ctx, G, d, T, base):
    """Blocks bit for bit, read back exactly; the rows before and behind stay as they were."""
    print(f"[case] kv4 append G={G} d={d} T={T} base={base}", flush=True)
    row, tail = G * d, 37
    n = base + T + tail
    old, new = F.normal(82, "old", n * row).reshape(n, row), F.normal(82, "new", T * row, 3.0).reshape(T, row)
    if T >= 8:
        new[:8] = _special_rows(row)
    kv = V.KVCache(ctx, 2, n + 3, G, d, V.KV_Q4_0)
    d_old, d_new = ctx.to_device(old), ctx.to_device(new)
    kv.append(1, d_old, d_old, n)
    kv.truncate(1, base)
    assert kv.used(1) == base
    kv.append(1, d_new, d_new, T)
    assert kv.used(1) == base + T and kv.used(0) == 0
    want = old.copy()
    want[base:base + T] = new
    blocks = F.quantize(want, V.DT_Q4_0).reshape(n, row // 32, 18)
    k, v, ks, vs = kv.read(1, 0, n)
    assert ks is None and vs is None
    assert np.array_equal(k, blocks) and np.array_equal(v, blocks)
    first = base // 2                                   # a part of the rows, from the middle of a group
    k, v, _, _ = kv.read(1, first, T)
    assert np.array_equal(k, blocks[first:first + T]) and np.array_equal(v, k)
    out = [ctx.to_device(np.full((n + 1, row), 7, np.float32)) for _ in range(2)]
    kv.dequant_into(1, n, *out)
    values = F.dequantize(blocks, V.DT_Q4_0, n * row).reshape(n, row)
    for o in out:
        got = o.download((n + 1, row))
        assert np.array_equal(got[:n], values) and (got[n:] == 7).all()
    assert not kv.read(0, 0, n)[0].any()                # the other layer
    kv.reset()
    assert kv.used(1) == 0 and not kv.read(1, 0, n + 3)[1].any()


def test_append_of_no_numbers(ctx):
    """A block with an infinity or a NaN reads back as NaN; its neighbours are as without it."""
    x = F.normal(83, "x", 40 * 128).reshape(40, 128)
    clean = F.dequantize(F.quantize(x, V.DT_Q4_0), V.DT_Q4_0, x.size).reshape(40, 4, 32)
    bad = x.copy()
    bad[3, 40], bad[4, 127], bad[39, 0] = np.nan, np.inf, -np.inf
    bad[20, 64:96] = 1e6                                # finite, its scale is not
    kv = V.KVCache(ctx, 1, 40, 1, 128, V.KV_Q4_0)
    kv.append(0, ctx.to_device(bad), ctx.to_device(bad), 40)
    outs = [ctx.alloc(x.nbytes) for _ in range(2)]
    kv.dequant_into(0, 40, *outs)
    for o in outs:
        got = o.download((40, 4, 32))
        where = np.zeros((40, 4), bool)
        where[[3, 4, 39, 20], [1, 3, 0, 2]] = True
        assert np.isnan(got[where]).all() and np.array_equal(got[~where], clean[~where])


@pytest.mark.parametrize("H,G,d,n,scale", [
    (4, 1, 64, 1, 0.125), (4, 4, 64, 2, 0.125), (32, 4, 64, 31, 0.125), (32, 4, 64, 32, 0.125), (8, 8, 128, 33, 0.1),
    (32, 8, 128, 127, 0.1), (32, 8, 128, 128, 0.1), (32, 4, 64, 129, 0.125), (24, 8, 64, 500, 0.125), (28, 4, 128, 777, 0.1),
    (16, 1, 64, 1000, 0.125), (17, 1, 128, 333, 0.1), (40, 1, 64, 2049, 0.125), (32, 8, 128, 4097, -0.1), (32, 4, 64, 4096, 0.0),
    (6, 2, 64, 9001, 0.125), (32, 8, 128, 6001, 1.5), (4, 1, 64, 40011, 0.125),
    (256, 256, 64, 100, 0.125), (250, 250, 128, 300, 0.1),
    (64, 1, 128, 40001, 0.1), (24, 1, 64, 40001, 0.125)])
def test_decode_attention(ctx, H, G, d, n, scale):
    """All group sizes, edges of the groups of keys; rows behind the context hold NaN; the call that
    allocates nothing gives the same bits, and so does a second call."""
    print(f"[case] kv4 decode H={H} G={G} d={d} n={n} scale={scale}", flush=True)
    kv, K, Vv = _filled(ctx, n, G, d, 84 + n, layers=2)
    big = V.KVCache(ctx, 1, n + 45, G, d, V.KV_Q4_0)    # the same rows, with others behind them
    k, v, _, _ = kv.read(1, 0, n)
    row = G * d
    pad = np.full((45, row), np.nan, np.float32)
    big.append(0, ctx.to_device(np.concatenate([K.reshape(n, row), pad])), ctx.to_device(np.concatenate([Vv.reshape(n, row), pad])), n + 45)
    q = F.normal(85, f"q{n}", H * d)
    dq, out, fix = ctx.to_device(q), ctx.to_device(np.full(H * d + 5, 7, np.float32)), ctx.alloc(q.nbytes)
    kv.attention_decode(1, dq, out, H, n, scale)
    got = out.download((H * d + 5,))
    ref, bound = _attention64(q.reshape(1, H, d), K, Vv, H, np.float32(scale))
    err = np.abs(got[:H * d].reshape(1, H, d) - ref)
    print(f"  largest error / bound {np.max(err / bound):.3g}", flush=True)
    assert (err <= bound).all() and (got[H * d:] == 7).all()
    kv.attention_decode(1, dq, out, H, n, scale)
    assert np.array_equal(out.download((H * d,)), got[:H * d])
    if H * ((n + 63) // 64) * (d + 2) <= 1 << 19:
        V.check(V.lib().vlrf_hip_attn_decode_noalloc(kv.h, 1, dq.ptr, fix.ptr, H, n, float(scale)))
        assert np.array_equal(fix.download((H * d,)), got[:H * d])
    # The re-quantized values may differ from the first cache's: compared with their own.
    Kb, Vb = ctx.alloc(n * row * 4), ctx.alloc(n * row * 4)
    big.dequant_into(0, n, Kb, Vb)
    big.attention_decode(0, dq, out, H, n, scale)
    ref, bound = _attention64(q.reshape(1, H, d), Kb.download((n, G, d)), Vb.download((n, G, d)), H, np.float32(scale))
    assert (np.abs(out.download((1, H, d)) - ref) <= bound).all()


@pytest.mark.parametrize("H,G,d,T,n,scale", [
    (4, 1, 64, 1, 1, 0.125), (4, 1, 64, 2, 2, 0.125), (8, 8, 64, 5, 5, 0.125), (32, 8, 128, 5, 300, 0.1),
    (24, 8, 64, 7, 33, 0.125), (28, 4, 128, 11, 40, 0.1), (32, 4, 64, 33, 33, 0.125), (32, 4, 64, 32, 64, -0.125),
    (8, 2, 128, 64, 64, 0.1), (16, 8, 64, 65, 200, 0.125), (17, 1, 64, 31, 95, 0.125), (32, 8, 128, 100, 1000, 0.1),
    (4, 4, 128, 257, 300, 0.1), (8, 2, 64, 300, 1029, 0.125), (4, 1, 64, 700, 700, 0.125), (12, 4, 128, 129, 3001, 0.1),
    (32, 8, 128, 1, 5000, 0.1), (32, 4, 64, 3, 9000, 0.125), (8, 8, 128, 513, 513, 2.0), (2, 1, 128, 1500, 1500, 0.1),
    (256, 256, 64, 3, 100, 0.125), (128, 128, 64, 129, 200, 0.125), (128, 128, 64, 127, 200, 0.125), (4, 4, 128, 4, 300, 0.1),
    (32, 8, 128, 13, 3001, 0.1), (16, 1, 64, 21, 12001, 0.125), (32, 8, 128, 5, 6001, 0.1), (32, 8, 128, 33, 700, 0.1),
    (128, 128, 64, 200, 333, 0.125), (128, 64, 128, 150, 333, -0.1), (256, 64, 128, 150, 333, -0.1), (64, 64, 128, 300, 301, 0.1)])
def test_chunk_attention(ctx, H, G, d, T, n, scale):
    """Chunks from one row on: ragged ones, groups of keys on the diagonal, few rows behind many keys."""
    print(f"[case] kv4 chunk H={H} G={G} d={d} T={T} n={n} scale={scale}", flush=True)
    kv, K, Vv = _filled(ctx, n, G, d, 86 + n, more=13)
    q = F.normal(87, f"q{T}", T * H * d).reshape(T, H, d)
    out = ctx.to_device(np.full(T * H * d + 5, 7, np.float32))
    kv.attention_chunk(0, ctx.to_device(q), out, H, T, n, scale)
    got = out.download((T * H * d + 5,))
    ref, bound = _attention64(q, K, Vv, H, np.float32(scale))
    err = np.abs(got[:-5].reshape(ref.shape) - ref)
    print(f"  largest error / bound {np.max(err / bound):.3g}", flush=True)
    assert (err <= bound).all() and (got[-5:] == 7).all()


@pytest.mark.parametrize("H,G,d,T,n", [(8, 2, 64, 40, 100), (4, 1, 128, 150, 150), (8, 2, 128, 300, 400), (2, 2, 64, 3, 70),
                                         (8, 2, 64, 600, 700), (128, 128, 64, 200, 333), (128, 64, 128, 150, 333), (256, 64, 128, 150, 333)])
def test_chunk_attention_masked_no_numbers(ctx, H, G, d, T, n):
    """A key or a value that is no number reaches the rows that see it and no other: the others
    are as far from the 64-bit result as they may be without it."""
    print(f"[case] kv4 masked NaN H={H} G={G} d={d} T={T} n={n}", flush=True)
    row = G * d
    K, Vv = (F.normal(88, c, n * row).reshape(n, row) for c in "kv")
    q = ctx.to_device(F.normal(88, "q", T * H * d))
    got = {}
    for name, at in (("none", None), ("k", (K, n - T + 1)), ("v", (Vv, n - T + 2)), ("first", (Vv, 0))):
        kv = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
        Kx, Vx = K.copy(), Vv.copy()
        if at is not None:
            (Kx if at[0] is K else Vx)[at[1], ::3] = np.inf if name == "k" else np.nan
        kv.append(0, ctx.to_device(Kx), ctx.to_device(Vx), n)
        out = ctx.alloc(T * H * d * 4)
        kv.attention_chunk(0, q, out, H, T, n, 0.1)
        got[name] = out.download((T, H * d))
    assert np.isfinite(got["none"]).all()
    # Groups of keys with such a scale come last, so sums may run in another order: each result
    # is within the same distance of the exact one.
    ref, bound = _attention64(q.download((T, H, d)), _decoded(K, n, G, d), _decoded(Vv, n, G, d), H, np.float32(0.1))
    for name, rows in (("none", T), ("k", 1), ("v", 2)):
        assert (np.abs(got[name].reshape(ref.shape) - ref) <= bound)[:rows].all(), name
        assert np.isnan(got[name][rows:]).all(), name
    assert np.isnan(got["first"]).all()


@pytest.mark.parametrize("H,G,T", [(8, 2, 1), (8, 2, 3), (8, 2, 200), (128, 64, 150), (256, 64, 150)])
@pytest.mark.parametrize("k_std,v_std", [(1.0, 5e4), (300.0, 1.0), (1.0, 1e-4), (1e-3, 30.0), (2e4, 2e4)])
def test_ranges_of_the_cache(ctx, k_std, v_std, H, G, T):
    """Scales up to f16's largest and small ones, side by side in one group of keys."""
    print(f"[case] kv4 ranges k={k_std} v={v_std} H={H} T={T}", flush=True)
    d, n = 128, 300
    row = G * d
    K, Vv = F.normal(89, "k", n * row, k_std).reshape(n, row), F.normal(89, "v", n * row, v_std).reshape(n, row)
    if v_std > 10:                                      # a block of usual values beside the large ones
        Vv[:, 32:64] *= 1 / v_std
        Vv[100:200] *= 1e-3
    kv = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
    kv.append(0, ctx.to_device(K), ctx.to_device(Vv), n)
    q = F.normal(89, "q", T * H * d).reshape(T, H, d)
    out = ctx.alloc(q.nbytes)
    scale = np.float32(0.1 / max(1.0, k_std))
    kv.attention_chunk(0, ctx.to_device(q), out, H, T, n, scale)
    ref, bound = _attention64(q, _decoded(K, n, G, d), _decoded(Vv, n, G, d), H, scale)
    assert (np.abs(out.download(q.shape) - ref) <= bound).all()


def test_ranges_of_queries(ctx):
    """Queries of very different sizes in one chunk, one of zeros (the mean of its keys), one with an infinity."""
    H, G, d, T, n = 8, 2, 64, 40, 77
    kv, K, Vv = _filled(ctx, n, G, d, 90)
    q = F.normal(90, "q", T * H * d).reshape(T, H, d)
    q[1], q[2], q[3], q[4, :, 5] = 0, q[2] * 1e-30, q[3] * 1e-41, q[4, :, 5] * 1e4
    clean = q.copy()
    q[5, 2, 7], q[6, 3, 0] = np.inf, np.nan
    out = ctx.alloc(q.nbytes)
    kv.attention_chunk(0, ctx.to_device(q), out, H, T, n, 0.125)
    got = out.download(q.shape)
    ref, bound = _attention64(clean, K, Vv, H, np.float32(0.125))
    bad = np.zeros((T, H), bool)
    bad[5, 2] = bad[6, 3] = True
    assert np.isnan(got[bad]).all()
    assert (np.abs(got - ref) <= bound)[~bad].all()


@pytest.mark.parametrize("G,rep,d,T", [(64, 8, 64, 3), (128, 1, 128, 2), (16, 16, 128, 60)])
def test_pieces_add_up(ctx, G, rep, d, T):
    """Queries with one element that is not zero, few keys: nothing but the two pieces of q and of the
    weights rounds, and a piece that does not fit the other (2^-11 off) stands out."""
    print(f"[case] kv4 pieces G={G} rep={rep} d={d} T={T}", flush=True)
    H = G * rep
    kv, K, Vv = _filled(ctx, T, G, d, 99)
    q = np.zeros((T, H, d), np.float32)
    at = np.arange(T * H)
    q.reshape(T * H, d)[at, at * 7 % d] = F.normal(99, "q", T * H, 4.0)
    out = ctx.alloc(q.nbytes)
    kv.attention_chunk(0, ctx.to_device(q), out, H, T, T, 1.0)
    ref, bound = _attention64(q, K, Vv, H, np.float32(1.0), terms=1)
    assert (np.abs(out.download(q.shape) - ref) <= bound).all()


def test_one_token_is_the_decode_call(ctx):
    kv, _, _ = _filled(ctx, 1500, 4, 64, 91)
    q = ctx.to_device(F.normal(91, "q", 32 * 64))
    a, b = ctx.alloc(8192), ctx.alloc(8192)
    kv.attention_decode(0, q, a, 32, 1500, 0.125)
    kv.attention_chunk(0, q, b, 32, 1, 1500, 0.125)
    assert np.array_equal(a.download((2048,)), b.download((2048,)))


def test_addresses_of_floats(ctx):
    """Rows, queries and results at addresses that are multiples of 4 only."""
    H, G, d, T, n = 8, 2, 64, 37, 90
    row = G * d
    K, Vv, q = F.normal(92, "k", n * row), F.normal(92, "v", n * row), F.normal(92, "q", T * H * d)

    class At:
        def __init__(self, a, more=0):
            self.buf = ctx.to_device(np.concatenate([np.zeros(1, np.float32), a, np.full(more, 7, np.float32)]))
            self.ptr = self.buf.ptr + 4

    kv = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
    kv.append(0, At(K), At(Vv), n)
    out = At(np.zeros(q.size, np.float32), 3)
    kv.attention_chunk(0, At(q), out, H, T, n, 0.125)
    got = out.buf.download((q.size + 4,))
    ref, bound = _attention64(q.reshape(T, H, d), _decoded(K.reshape(n, row), n, G, d), _decoded(Vv.reshape(n, row), n, G, d), H,
                              np.float32(0.125))
    assert (np.abs(got[1:-3].reshape(T, H, d) - ref) <= bound).all() and got[0] == 0 and (got[-3:] == 7).all()
    ko, vo = At(np.zeros(n * row, np.float32), 3), At(np.zeros(n * row, np.float32), 3)
    kv.dequant_into(0, n, ko, vo)
    got = ko.buf.download((n * row + 4,))
    assert np.array_equal(got[1:-3], _decoded(K.reshape(n, row), n, G, d).ravel()) and got[0] == 0 and (got[-3:] == 7).all()


def test_heads_past_32_bits(ctx):
    """Heads whose codes begin past 4 GiB."""
    G, d, cap, n = 70, 128, 1 << 20, 45
    print(f"[case] kv4 offsets: {G} heads of {cap} rows", flush=True)
    row = G * d
    K, Vv = F.normal(93, "k", n * row).reshape(n, row), F.normal(93, "v", n * row).reshape(n, row)
    kv = V.KVCache(ctx, 1, cap, G, d, V.KV_Q4_0)
    kv.append(0, ctx.to_device(K), ctx.to_device(Vv), n)
    for T in (1, 9):
        q = F.normal(93, "q", T * G * d).reshape(T, G, d)
        out = ctx.alloc(q.nbytes)
        kv.attention_chunk(0, ctx.to_device(q), out, G, T, n, 0.1)
        ref, bound = _attention64(q, _decoded(K, n, G, d), _decoded(Vv, n, G, d), G, np.float32(0.1))
        assert (np.abs(out.download(q.shape) - ref) <= bound).all()
    blocks, _, _, _ = kv.read(0, 0, n)
    assert np.array_equal(blocks.ravel(), F.quantize(K, V.DT_Q4_0))
    ko, vo = ctx.alloc(K.nbytes), ctx.alloc(K.nbytes)
    kv.dequant_into(0, n, ko, vo)
    assert np.array_equal(vo.download((n, G, d)), _decoded(Vv, n, G, d))


def test_prompt_in_chunks_then_tokens(ctx):
    """As a program uses them together: a prompt appended and attended in chunks, tokens one by one,
    drafted tokens of which some are taken back; each result against 64 bits over what was there."""
    H, G, d, cap = 16, 4, 64, 400
    row, scale = G * d, np.float32(0.125)
    K, Vv = F.normal(94, "k", cap * row).reshape(cap, row), F.normal(94, "v", cap * row).reshape(cap, row)
    Kd, Vd = _decoded(K, cap, G, d), _decoded(Vv, cap, G, d)
    kv = V.KVCache(ctx, 1, cap, G, d, V.KV_Q4_0)
    at = 0
    for step, (T, keep) in enumerate([(150, 150), (77, 77), (1, 1), (1, 1), (6, 2), (1, 1), (5, 5), (100, 64), (1, 1)]):
        kv.append(0, ctx.to_device(K[at:at + T]), ctx.to_device(Vv[at:at + T]), T)
        n = at + T
        assert kv.used(0) == n
        q = F.normal(95 + step, "q", T * H * d).reshape(T, H, d)
        out, dq = ctx.alloc(q.nbytes), ctx.to_device(q)
        if T == 1:
            kv.attention_decode(0, dq, out, H, n, scale)
        else:
            kv.attention_chunk(0, dq, out, H, T, n, scale)
        ref, bound = _attention64(q, Kd[:n], Vd[:n], H, scale)
        assert (np.abs(out.download(q.shape) - ref) <= bound).all(), (step, n)
        at += keep
        kv.truncate(0, at)


def test_captured_and_replayed():
    """Decode and chunk calls captured into one graph: replays, with eager calls of other sizes
    between them, give the eager result; a call whose scratch would have to grow is refused while
    the stream is captured."""
    from test_gpu_prefill_gemm import _hip
    hip, ctx = _hip(), V.Context(0)
    H, G, d, n = 32, 8, 128, 3000
    row = G * d
    kv = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
    rows = [ctx.to_device(F.normal(96, c, n * row)) for c in "kv"]
    kv.append(0, rows[0], rows[1], n - 60)
    q = ctx.to_device(F.normal(96, "q", 300 * H * d))
    outs = [ctx.alloc(300 * H * d * 4) for _ in range(3)]

    def calls():
        V.check(V.lib().vlrf_hip_kv_append(kv.h, 0, rows[0].ptr, rows[1].ptr, 40))
        V.check(V.lib().vlrf_hip_attn_decode(kv.h, 0, q.ptr, outs[0].ptr, H, n - 20, C.c_float(0.1)))
        V.check(V.lib().vlrf_hip_attn_chunk(kv.h, 0, q.ptr, outs[1].ptr, H, 40, n - 20, C.c_float(0.1)))
        V.check(V.lib().vlrf_hip_attn_chunk(kv.h, 0, q.ptr, outs[2].ptr, H, 300, n - 20, C.c_float(0.1)))

    sizes = [(H * d,), (40 * H * d,), (300 * H * d,)]
    calls()
    eager = [o.download(s) for o, s in zip(outs, sizes)]
    kv.truncate(0, n - 60)
    s, g, ge = C.c_void_p(ctx.stream()), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(s, 2) == 0
    try:
        calls()
    finally:
        rc = hip.hipStreamEndCapture(s, C.byref(g))
    assert rc == 0
    assert hip.hipGraphInstantiate(C.byref(ge), g, None, None, 0) == 0
    other = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
    other.append(0, rows[1], rows[0], n)
    scrap = ctx.alloc(300 * H * d * 4)
    for i in range(3):
        for o in outs:
            o.zero()
        other.attention_decode(0, q, scrap, H, n - 7 * i, 0.1)
        other.attention_chunk(0, q, scrap, H, 300 - 50 * i, n - 7 * i, 0.1)
        assert hip.hipGraphLaunch(ge, s) == 0
        other.attention_chunk(0, q, scrap, H, 12, n, 0.1)
        ctx.sync()
        for o, size, want in zip(outs, sizes, eager):
            assert np.array_equal(o.download(size), want)
    hip.hipGraphExecDestroy(ge)
    hip.hipGraphDestroy(g)


def test_two_contexts_at_once(ctx):
    """Calls queued on two contexts' streams without a wait between them."""
    other = V.Context(0)
    H, G, d, n = 32, 4, 64, 5000
    jobs = []
    for c, seed in ((ctx, 97), (other, 98)):
        kv, K, Vv = _filled(c, n, G, d, seed)
        q = F.normal(seed, "q", 3 * H * d).reshape(3, H, d)
        jobs.append((c, kv, q, c.to_device(q), c.alloc(q.nbytes), _attention64(q, K, Vv, H, np.float32(0.125))))
    for _ in range(20):
        for _, kv, _, dq, out, _ in jobs:
            kv.attention_chunk(0, dq, out, H, 3, n, 0.125)
    for c, _, q, _, out, (ref, bound) in jobs:
        c.sync()
        assert (np.abs(out.download(q.shape) - ref) <= bound).all()


def test_refusals(ctx):
    lib = V.lib()
    for d in (16, 48, 80):
        with pytest.raises(V.HipError, match="whole Q4_0 blocks"):
            V.KVCache(ctx, 1, 8, 2, d, V.KV_Q4_0)
    with pytest.raises(V.HipError, match="cache dtype 4"):
        V.KVCache(ctx, 1, 8, 2, 64, 4)
    kv = V.KVCache(ctx, 1, 50, 2, 64, V.KV_Q4_0)
    x, out = ctx.to_device(np.zeros(60 * 128, np.float32)), ctx.alloc(60 * 128 * 4)
    kv.append(0, x, x, 30)
    for T, rc in ((21, _lib.ERR_OVERFLOW), (2 ** 31 - 1, _lib.ERR_OVERFLOW), (0, _lib.ERR_ARG), (-1, _lib.ERR_ARG)):
        assert lib.vlrf_hip_kv_append(kv.h, 0, x.ptr, x.ptr, T) == rc and kv.used(0) == 30
    for n in (-1, 31):
        assert lib.vlrf_hip_kv_truncate(kv.h, 0, n) == _lib.ERR_ARG and kv.used(0) == 30
    assert lib.vlrf_hip_kv_truncate(kv.h, 1, 0) == _lib.ERR_ARG

    def chunk(h=kv.h, layer=0, q=x.ptr, o=out.ptr, heads=4, T=3, n=30):
        return lib.vlrf_hip_attn_chunk(h, layer, q, o, heads, T, n, C.c_float(0.1))

    assert chunk() == 0
    for o in (out.ptr, out.ptr + 4, out.ptr + 3 * 4 * 64 * 4 - 4):   # q and out side by side, not over each other
        assert chunk(q=out.ptr, o=o) == _lib.ERR_ARG and "overlap" in _lib.last_error()
        assert chunk(q=o, o=out.ptr) == _lib.ERR_ARG
    assert chunk(q=x.ptr, o=x.ptr + 3 * 4 * 64 * 4) == 0
    for bad in (dict(layer=1), dict(layer=-1), dict(q=None), dict(o=None), dict(o=x.ptr), dict(heads=3), dict(heads=0),
                dict(heads=-2), dict(T=0), dict(T=31), dict(T=-1), dict(n=51), dict(n=0), dict(n=2), dict(n=-5)):
        assert chunk(**bad) == _lib.ERR_ARG, bad
        assert _lib.last_error()
    for bad in (dict(n_heads=3), dict(n=0), dict(n=51), dict(n_heads=0), dict(n_heads=-4)):
        a = dict(n_heads=4, n=30, **{}) | bad
        for fn in (lib.vlrf_hip_attn_decode, lib.vlrf_hip_attn_decode_noalloc):
            assert fn(kv.h, 0, x.ptr, out.ptr, a["n_heads"], a["n"], C.c_float(0.1)) == _lib.ERR_ARG, bad
    q8 = V.KVCache(ctx, 1, 50, 2, 64, V.KV_Q8_0)
    assert chunk(h=q8.h) == _lib.ERR_ARG and "not Q4_0" in _lib.last_error()
    wide = V.KVCache(ctx, 1, 50, 2, 96, V.KV_Q4_0)       # appended and read back, not attended
    wide.append(0, x, x, 30)
    assert chunk(h=wide.h) == _lib.ERR_ARG and "d_head 96" in _lib.last_error()
    ctx.sync()


@pytest.mark.parametrize("d", [32, 160, 256, 512, 544, 1024, 2048])
def test_refused_d_head_of_attention(ctx, d):
    """A cache of any whole number of blocks a row is appended to and read back; attention over it is an
    error, whatever the size, by each of the three calls."""
    print(f"[case] kv4 refused d_head={d}", flush=True)
    H, G, n = 4, 1, 100
    lib = V.lib()
    kv = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
    x = ctx.to_device(F.normal(100, "wide", n * d))
    q, out = ctx.to_device(np.zeros(3 * H * d, np.float32)), ctx.to_device(np.full(3 * H * d, 7, np.float32))
    kv.append(0, x, x, n)
    for rc in (lib.vlrf_hip_attn_decode(kv.h, 0, q.ptr, out.ptr, H, n, C.c_float(0.1)),
               lib.vlrf_hip_attn_decode_noalloc(kv.h, 0, q.ptr, out.ptr, H, n, C.c_float(0.1)),
               lib.vlrf_hip_attn_chunk(kv.h, 0, q.ptr, out.ptr, H, 3, n, C.c_float(0.1))):
        assert rc == _lib.ERR_ARG and f"d_head {d}" in _lib.last_error()
    assert (out.download((3 * H * d,)) == 7).all()
    assert np.array_equal(kv.read(0, 0, n)[1].ravel(), F.quantize(x.download((n, d)), V.DT_Q4_0))


@pytest.mark.parametrize("H,G,d,n", [(32, 8, 128, 8065), (32, 8, 128, 120001), (32, 4, 64, 30011), (15, 1, 128, 65600),
                                     (16, 1, 64, 65600)])
def test_decode_without_allocation_over_long_contexts(H, G, d, n):
    """The call that allocates nothing at contexts where the other caches' partials would not fit, the
    first call of its context and captured: the bits of the call with scratch."""
    print(f"[case] kv4 noalloc H={H} G={G} d={d} n={n}", flush=True)
    from test_gpu_prefill_gemm import _hip
    hip, ctx, lib = _hip(), V.Context(0), V.lib()
    assert H * ((n + 63) // 64) * (d + 2) > 1 << 19
    row = G * d
    x = ctx.to_device(F.normal(101, "rows", n * row))
    kv = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
    kv.append(0, x, x, n)
    q, fix, out = ctx.to_device(F.normal(101, "q", H * d)), ctx.to_device(np.full(H * d + 5, 7, np.float32)), ctx.alloc(H * d * 4)
    V.check(lib.vlrf_hip_attn_decode_noalloc(kv.h, 0, q.ptr, fix.ptr, H, n, C.c_float(0.1)))
    got = fix.download((H * d + 5,))
    kv.attention_decode(0, q, out, H, n, 0.1)
    assert np.array_equal(got[:H * d], out.download((H * d,))) and (got[H * d:] == 7).all() and np.abs(got[:H * d]).max() > 0
    s, g, ge = C.c_void_p(ctx.stream()), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(s, 2) == 0
    try:
        rc = lib.vlrf_hip_attn_decode_noalloc(kv.h, 0, q.ptr, fix.ptr, H, n, C.c_float(0.1))
    finally:
        end = hip.hipStreamEndCapture(s, C.byref(g))
    assert rc == 0 and end == 0
    assert hip.hipGraphInstantiate(C.byref(ge), g, None, None, 0) == 0
    for i in range(3):
        fix.zero()
        kv.attention_decode(0, q, out, H, n - 1 - i, 0.1)
        assert hip.hipGraphLaunch(ge, s) == 0
        ctx.sync()
        assert np.array_equal(fix.download((H * d,)), got[:H * d])
    hip.hipGraphExecDestroy(ge)
    hip.hipGraphDestroy(g)


def test_decode_without_allocation_refuses_what_does_not_fit(ctx):
    """16 query heads of 128 on one KV head: 256 workgroups' partials are more than the fixed array."""
    H, n = 16, 65600
    x = ctx.to_device(F.normal(102, "rows", n * 128))
    kv = V.KVCache(ctx, 1, n, 1, 128, V.KV_Q4_0)
    kv.append(0, x, x, n)
    q, out = ctx.to_device(F.normal(102, "q", H * 128)), ctx.to_device(np.full(H * 128, 7, np.float32))
    for m in (65537, n):
        rc = V.lib().vlrf_hip_attn_decode_noalloc(kv.h, 0, q.ptr, out.ptr, H, m, C.c_float(0.1))
        assert rc == _lib.ERR_ARG and "exceed the fixed scratch" in _lib.last_error()
        assert (out.download((H * 128,)) == 7).all()
    assert V.lib().vlrf_hip_attn_decode_noalloc(kv.h, 0, q.ptr, out.ptr, H, 65536, C.c_float(0.1)) == 0
    got = out.download((H * 128,))
    kv.attention_decode(0, q, out, H, 65536, 0.1)
    assert np.array_equal(out.download((H * 128,)), got)


def test_scratch_does_not_grow_under_capture():
    """Calls whose partials need more scratch than the context holds are an error while its stream is
    captured, and the capture goes on; after the same call once before, they are recorded."""
    from test_gpu_prefill_gemm import _hip
    hip, ctx, lib = _hip(), V.Context(0), V.lib()
    H, G, d, n = 32, 8, 128, 3000
    x = ctx.to_device(F.normal(103, "rows", n * G * d))
    kv = V.KVCache(ctx, 1, n, G, d, V.KV_Q4_0)
    kv.append(0, x, x, n)
    q, outs = ctx.to_device(F.normal(103, "q", 5 * H * d)), [ctx.to_device(np.full(5 * H * d, 7, np.float32)) for _ in range(2)]
    s = C.c_void_p(ctx.stream())

    def calls():
        return [lib.vlrf_hip_attn_decode(kv.h, 0, q.ptr, outs[0].ptr, H, n, C.c_float(0.1)),
                lib.vlrf_hip_attn_chunk(kv.h, 0, q.ptr, outs[1].ptr, H, 5, n, C.c_float(0.1))]

    def captured():
        g = C.c_void_p()
        assert hip.hipStreamBeginCapture(s, 2) == 0
        try:
            rcs, said = calls(), _lib.last_error()
        finally:
            rc = hip.hipStreamEndCapture(s, C.byref(g))
        assert rc == 0
        return rcs, said, g

    rcs, said, g = captured()
    assert rcs == [_lib.ERR_ARG] * 2 and "captured" in said
    hip.hipGraphDestroy(g)
    assert all((o.download((5 * H * d,)) == 7).all() for o in outs)
    assert calls() == [0, 0]
    want = [o.download((5 * H * d,)) for o in outs]
    rcs, _, g = captured()
    assert rcs == [0, 0]
    ge = C.c_void_p()
    assert hip.hipGraphInstantiate(C.byref(ge), g, None, None, 0) == 0
    for i in range(3):
        for o in outs:
            o.zero()
        kv.attention_decode(0, q, outs[0], H, n - 1 - i, 0.1)
        assert hip.hipGraphLaunch(ge, s) == 0
        ctx.sync()
        got = [o.download((5 * H * d,)) for o in outs]
        assert np.array_equal(got[0][:H * d], want[0][:H * d]) and np.array_equal(got[1], want[1])
    hip.hipGraphExecDestroy(ge)
    hip.hipGraphDestroy(g)
