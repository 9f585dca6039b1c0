"""Models over the 4-bit KV cache (kv_dtype KV_Q4_0) against the same decoder in
64 bits with a cache that holds the same blocks: decode steps (one workgroup a
head group, and several that share the keys), the captured graph, the batched
prefill in chunks, and the rows that they leave in the cache."""
import numpy as np
import pytest

import vlrf_amd as V
from conftest import rel_err
from vlrf_amd import formats as F

pytestmark = pytest.mark.gpu


def _held(m, layer, n):
    """K and V rows [0, n) of a layer, [n, n_kv * d_head], and the scales of their blocks, as wide."""
    out = []
    for blocks in m.kv_rows(layer, 0, n)[:2]:
        scale = np.abs(blocks.reshape(n, -1, 18)[:, :, :2].copy().view(np.float16).astype(np.float64))
        out.append((F.dequantize(blocks, V.DT_Q4_0, blocks.size // 18 * 32).reshape(n, -1).astype(np.float64),
                    scale.repeat(32, 1).reshape(n, -1)))
    return out


def _check_held(held, scale, new, tol):
    """A code is the nearest of 16 multiples of the scale, the smallest -8, the largest 7: half a step off,
    one at the far end. The scale's own rounding moves a value by 8 * 2^-11 steps at most, an error tol of the
    K or V (of the largest) by as much; with it a value at a border takes the code on its other side, which is
    half a step off too."""
    off = np.abs(held - new)
    slack = tol * np.abs(new).max() + 2.0 ** -8 * scale
    assert (off <= scale + slack).all()
    far = np.abs(new) >= 7.4 * scale   # the far end, where the code 7 stands for up to 8 steps
    assert (off <= 0.5 * scale + slack)[~far].all()


class Decoder:
    """RMSNorm, half-split RoPE, GQA attention over stored K/V, SwiGLU, in 64 bits."""

    def __init__(self, cfg, weights):
        self.c, self.w = cfg, {k: np.asarray(v, np.float64) for k, v in weights.items()}
        self.H, self.G = cfg["n_heads"], cfg["n_kv_heads"]
        self.d = cfg["d_model"] // self.H
        i = np.arange(self.d // 2, dtype=np.float32)
        freq = np.float32(1) / np.power(np.float32(cfg["rope_theta"]), np.float32(2) * i / np.float32(self.d))
        angle = (np.arange(cfg["max_seq_len"], dtype=np.float32)[:, None] * freq).astype(np.float32)
        self.cos, self.sin = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c["norm_eps"]) * w

    def rope(self, x, pos):
        h = x.reshape(len(pos), -1, self.d)
        a, b = h[..., :self.d // 2], h[..., self.d // 2:]
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        return np.concatenate([a * c - b * s, b * c + a * s], -1).reshape(x.shape)

    def layers(self, x, stored):
        """x [T, d_model], the last T rows of the cache, through the layers; stored[layer] = (K, V): what the
        cache holds of all rows. Its own rows' K and V before they are stored: self.new[layer]."""
        T = x.shape[0]
        self.new = []
        for l in range(self.c["n_layers"]):
            w = lambda n: self.w[f"layers.{l}.{n}.weight"]   # noqa: E731
            K, Vs = stored[l]
            n = len(K)
            pos = n - T + np.arange(T)
            h = self.norm(x, w("ln1").ravel())
            q, k = self.rope(h @ w("attn.q_proj").T, pos), self.rope(h @ w("attn.k_proj").T, pos)
            v = h @ w("attn.v_proj").T
            self.new.append((k, v))
            keep = np.arange(n)[None] <= pos[:, None]
            out = np.empty_like(q)
            for hd in range(self.H):
                g, qs = hd // (self.H // self.G), slice(hd * self.d, (hd + 1) * self.d)
                ks = slice(g * self.d, (g + 1) * self.d)
                s = np.where(keep, q[:, qs] @ K[:, ks].T / np.sqrt(self.d), -np.inf)
                p = np.exp(s - s.max(1, keepdims=True))
                out[:, qs] = p @ Vs[:, ks] / p.sum(1, keepdims=True)
            x = x + out @ w("attn.o_proj").T
            h = self.norm(x, w("ln2").ravel())
            g = h @ w("ffn.gate").T
            x = x + (g / (1 + np.exp(-g)) * (h @ w("ffn.fc1").T)) @ w("ffn.fc2").T
        return x

    def logits(self, tok, stored):
        x = self.layers(self.w["embed.weight"][[tok]], stored)
        return (self.norm(x, self.w["ln_final.weight"].ravel()) @ self.w["lm_head.weight"].T)[0]


def _cfg(n_heads, n_kv, d_model, cap, n_layers=2, weight_dtype=V.DT_Q8_0):
    return dict(F.tiny(weight_dtype, n_layers=n_layers, max_seq_len=cap), n_heads=n_heads, n_kv_heads=n_kv,
                d_model=d_model, d_ff=2 * d_model if d_model <= 1024 else 512, kv_dtype=V.KV_Q4_0)


def _models(ctx, cfg, seed):
    m = V.Model(ctx, cfg)
    return m, Decoder(cfg, F.load_model(m, seed, want_f32=True, norm_std=0.1))


@pytest.mark.parametrize("n_heads,n_kv,d_model,cap,tokens,weights", [
    (4, 1, 256, 160, 40, V.DT_Q8_0), (4, 4, 256, 64, 40, V.DT_Q4_0), (8, 2, 1024, 300, 40, V.DT_Q8_0),
    (8, 8, 512, 1100, 300, V.DT_Q8_0), (8, 1, 1024, 700, 300, V.DT_Q4_0), (4, 2, 256, 80, 20, V.DT_F32),
    (4, 1, 256, 70000, 10, V.DT_Q8_0)])
def test_steps(ctx, n_heads, n_kv, d_model, cap, tokens, weights):
    """Logits of teacher-forced steps, and the rows they store, against the layers attending to what the cache
    holds (f32-class: 1e-3 of the largest). Not to blocks of the reference's own: a value within f32 rounding
    of a border between two codes may take the other, a whole step, which is no rounding of f32."""
    print(f"[case] kv4 model {n_heads}/{n_kv} d_model={d_model} cap={cap}", flush=True)
    cfg = _cfg(n_heads, n_kv, d_model, cap, weight_dtype=weights)
    m, ref = _models(ctx, cfg, 71)
    for i, t in enumerate(F.tokens(71, "kv4m", tokens, cfg["vocab_size"])):
        _, got = m.step(int(t), want_logits=True)
        if i < 8 or i % 16 == 0 or i == tokens - 1:
            held = [_held(m, layer, i + 1) for layer in range(cfg["n_layers"])]
            want = ref.logits(int(t), [(k[0], v[0]) for k, v in held])
            assert rel_err(got, want) <= 1e-3, i
            for layer in range(cfg["n_layers"]):
                for (h, scale), new in zip(held[layer], ref.new[layer]):
                    _check_held(h[i:], scale[i:], new, 1e-3)
    assert m.kv_rows(0, 0, 1)[2:] == (None, None)
    kv = m.step_bytes(100)[1]
    assert kv == cfg["n_layers"] * 2 * 100 * n_kv * (d_model // n_heads) * 18 / 32


@pytest.mark.parametrize("n_heads,n_kv,d_model,cap", [(4, 1, 256, 200), (8, 2, 1024, 1300)])
def test_generation_is_the_steps(ctx, monkeypatch, n_heads, n_kv, d_model, cap):
    """Greedy runs over captured graphs (one step, 16 steps), over launches one by one, step by step,
    and after a reset give the same ids; the graphs' positions run on across the calls."""
    cfg = _cfg(n_heads, n_kv, d_model, cap)
    m, _ = _models(ctx, cfg, 72)
    prompt = F.tokens(72, "kv4g", 30, cfg["vocab_size"])
    runs = [list(m.generate(prompt, 70)) for _ in range(2)]
    m.reset()
    m.prefill(prompt)
    tok, steps = int(prompt[-1]), []
    for _ in range(70):
        tok = m.step(tok)
        steps.append(tok)
    monkeypatch.setenv("VLRF_HIP_GRAPH", "0")
    m2, _ = _models(ctx, cfg, 72)
    assert runs[0] == runs[1] == steps == list(m2.generate(prompt, 70))
    assert m.used == 100
    m2.reset()
    kinds = m2.time_launches(5, 3)
    assert kinds["attn"][1] >= 2 * cfg["n_layers"] * 3 and "qkv_attn" in kinds


@pytest.mark.parametrize("n_heads,n_kv,d_model,cap,attn", [(4, 1, 256, 70000, 3), (8, 2, 1024, 300, 2)])
def test_every_launch_of_a_step_is_timed(ctx, n_heads, n_kv, d_model, cap, attn):
    """Append, attention and, where many workgroups share a KV head's keys, its merge; and what comes after."""
    cfg = _cfg(n_heads, n_kv, d_model, cap, n_layers=4)
    m = V.Model(ctx, cfg)
    F.load_model(m, 76)
    kinds = m.time_launches(5, 6)
    calls = {k: v[1] for k, v in kinds.items()}
    assert calls["attn"] == attn * 4 * 6 and calls["qkv_attn"] == calls["o_proj"] == calls["gate_up"] == calls["down"] == 4 * 6, calls


@pytest.mark.parametrize("n_heads,n_kv,d_model,chunks", [
    (4, 1, 256, (70, 45)), (8, 2, 1024, (1, 33, 90)), (8, 8, 512, (300, 20)), (8, 8, 512, (3900, 200)),
    (16, 2, 1024, (600,)), (32, 8, 2048, (1700,)), (32, 8, 4096, (1777, 30))])
def test_prefill_layer(ctx, n_heads, n_kv, d_model, chunks):
    """One layer over embedded rows in chunks (few rows, and enough for the many-rows kernel): the output
    in the bf16 class (1e-2) of the layer attending to what the cache holds, whose values are within half
    a step and that class of the layer's own K and V."""
    print(f"[case] kv4 prefill {n_heads}/{n_kv} d_model={d_model} chunks={chunks}", flush=True)
    total = sum(chunks)
    cfg = _cfg(n_heads, n_kv, d_model, total + 5, n_layers=1)
    m, ref = _models(ctx, cfg, 73)
    x = F.normal(73, "kv4x", total * d_model).reshape(total, d_model)
    at = 0
    for T in chunks:
        got = m.forward_hidden(ctx.to_device(x[at:at + T])).download((T, d_model))
        (K, k_scale), (Vs, v_scale) = _held(m, 0, at + T)
        want = ref.layers(x[at:at + T].astype(np.float64), [(K, Vs)])
        assert rel_err(got, want) <= 1e-2, at
        for held, scale, new in ((K, k_scale, ref.new[0][0]), (Vs, v_scale, ref.new[0][1])):
            _check_held(held[at:], scale[at:], new, 1e-2)
        at += T
    assert m.used == total


def test_prefill_then_steps(ctx):
    """A batched prefill, then decode steps over what it stored: close to the steps after a prefill one
    token at a time (the prompt's K and V differ in the bf16 class and, where that crosses a border, by a
    code)."""
    cfg = _cfg(8, 2, 512, 200)
    m, _ = _models(ctx, cfg, 74)
    prompt = F.tokens(74, "kv4p", 90, cfg["vocab_size"])
    out = []
    for prefill in (m.prefill, m.prefill_mfma):
        m.reset()
        prefill(prompt)
        assert m.used == 90
        out.append([m.step(int(t), want_logits=True)[1] for t in prompt[:5]])
    for a, b in zip(*out):
        assert np.isfinite(b).all() and rel_err(b, a) <= 0.1


def test_refusals(ctx):
    with pytest.raises(V.HipError, match="KV cache dtype 4"):
        V.Model(ctx, dict(F.tiny(), kv_dtype=4))
    m = V.Model(ctx, _cfg(4, 1, 256, 20, n_layers=1))
    F.load_model(m, 75)
    m.prefill(F.tokens(75, "r", 20, 512))
    for call in (lambda: m.step(1), lambda: m.prefill_mfma([1]), lambda: m.generate_async(1, 1)):
        with pytest.raises(V.HipError, match="exceeds max_seq_len"):
            call()
    assert m.used == 20
