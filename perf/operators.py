"""What the operators of the 4-bit KV cache (KV_Q4_0) are measured on: the calls
a program makes of them, from one token to a long context.

  write    KVCache.append, then dequant_into: T rows quantized behind `base`
           earlier ones, and the cache's rows read back.
  read     KVCache.dequant_into: a filled cache read back.
  decode   KVCache.attention_decode: one token's attention over the cache.
  chunk    KVCache.attention_chunk: causal attention of the cache's last T rows.

The cache holds Q4_0 blocks: 32 elements of a head's row share the f16 scale
d = max / -8 (max: the element of largest magnitude, the first of equal ones),
and an element is the code clamp(int(x * (1 / d) + 8.5), 0, 15), each operation
rounded to f32, standing for (code - 8) * d.  `own` false: the same in elementary
torch operations on blocks kept token by token (two codes a byte, even element
in the low half).
"""
import math
import zlib

import torch

own = False

# The head layouts of the benchmarks' decoder shapes (1.1B: 32/4 heads of 64, 8B: 32/8 of 128, tiny: 4/1 of 64).
LAYOUTS = {"1.1B": (32, 4, 64), "8B": (32, 8, 128), "tiny": (4, 1, 64)}


def _case(name, op, layout, **sizes):
    H, G, d = LAYOUTS[layout]
    return dict(name=name, op=op, H=H, G=G, d=d, **sizes)


def listed():
    return [
        # The token of a decode step, quantized into an empty cache: the smallest call, bound by latency.
        _case("write_1_row_tiny", "write", "tiny", base=0, T=1),
        # A later chunk of a prompt, at a row that is no multiple of anything.
        _case("write_333_at_517_1b", "write", "1.1B", base=517, T=333),
        # A long prompt at once.
        _case("write_16000_8b", "write", "8B", base=0, T=16000),
        # A cache read back at the length of the attention benchmark.
        _case("read_4096_1b", "read", "1.1B", ctx=4096),
        # A long context read back.
        _case("read_30001_8b", "read", "8B", ctx=30001),
        # Decode attention early in a conversation.
        _case("decode_200_1b", "decode", "1.1B", ctx=200),
        # At the length of the attention benchmark.
        _case("decode_4096_1b", "decode", "1.1B", ctx=4096),
        # A long conversation.
        _case("decode_15001_8b", "decode", "8B", ctx=15001),
        # The long contexts that a 4-bit cache is for.
        _case("decode_120001_8b", "decode", "8B", ctx=120001),
        # Drafted tokens checked together behind a conversation.
        _case("chunk_5_of_3001_8b", "chunk", "8B", T=5, ctx=3001),
        # A short prompt's second half.
        _case("chunk_233_of_700_1b", "chunk", "1.1B", T=233, ctx=700),
        # A long prompt's later chunk.
        _case("chunk_1777_of_4001_8b", "chunk", "8B", T=1777, ctx=4001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk"])
    # The shapes' layouts, a layout without shared heads, and groups of 2, 3 and 7 query heads.
    H, G, d = rng.choice([(32, 4, 64), (32, 8, 128), (32, 8, 128), (8, 8, 64), (16, 8, 64), (24, 8, 128), (28, 4, 128), (4, 1, 64)])
    case = dict(op=op, H=H, G=G, d=d)
    if op == "write":
        return dict(case, base=rng.choice([0, 0, _log(rng, 1, 4000)]), T=_log(rng, 1, 12000))
    if op == "read":
        return dict(case, ctx=_log(rng, 1, 30001))
    if op == "decode":
        return dict(case, ctx=_log(rng, 1, 120001))
    T = _log(rng, 1, 1777)
    return dict(case, T=T, ctx=T + rng.choice([0, _log(rng, 1, 2200)]))


# ---- inputs ------------------------------------------------------------------
def _normal(seed, name, shape):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + zlib.crc32(name.encode())) & 0x7FFFFFFFFFFF)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(seed, name, n, width):
    """n rows of keys or values: keys have a few channels that are several times as large as the others."""
    x = _normal(seed, name, (n, width))
    if name.startswith("k"):
        x.mul_(torch.where(_normal(seed, name + ".channels", (width,)).abs() > 2.2, 6.0, 1.0))
    return x


def _inputs(case, seed):
    """(earlier or all rows of the cache, rows to append, queries) of a case, f32; None where it has none."""
    H, G, d = case["H"], case["G"], case["d"]
    if case["op"] == "write":
        base, T = case["base"], case["T"]
        old = (_rows(seed, "k.old", base, G * d), _rows(seed, "v.old", base, G * d)) if base else None
        return old, (_rows(seed, "k.new", T, G * d), _rows(seed, "v.new", T, G * d)), None
    n = case["ctx"]
    rows = (_rows(seed, "k", n, G * d), _rows(seed, "v", n, G * d))
    if case["op"] == "read":
        return rows, None, None
    T = case.get("T", 1)
    return rows, None, _normal(seed, "q", (T, H * d))


class _Buffer:
    """A torch tensor as the binding takes buffers: its device address and size."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


_CONTEXT = []


def _context():
    import vlrf_amd as V
    if not _CONTEXT:                   # one context for the program, as a server keeps it
        _CONTEXT.append(V.Context(0))
    return _CONTEXT[0]


def _handle(case, old):
    """The framework's cache with the rows that are in it before the call."""
    import vlrf_amd as V
    n = case["base"] + case["T"] if case["op"] == "write" else case["ctx"]
    cache = V.KVCache(_context(), 1, n, case["G"], case["d"], dtype=V.KV_Q4_0)
    if old is not None:
        cache.append(0, _Buffer(old[0]), _Buffer(old[1]), old[0].shape[0])
    return cache


def prepare(case, seed):
    if not own:
        return _prepare(case, seed)
    # The context's stream is not ordered with torch's: inputs are made on it, and outputs belong to
    # it, so that the calls come after the inputs and no tensor is used again before they are done.
    with torch.cuda.stream(torch.cuda.ExternalStream(_context().stream())):
        return _prepare(case, seed)


def _prepare(case, seed):
    old, new, q = _inputs(case, seed)
    n = case["base"] + case["T"] if case["op"] == "write" else case["ctx"]
    width = case["G"] * case["d"]
    state = {"case": case, "new": new, "q": q}
    if own:
        state["cache"] = _handle(case, old)
    else:
        state["old"] = None if old is None else tuple(_blocks(x) for x in old)
    if q is None:
        state["out"] = [torch.empty(n, width, device="cuda") for _ in range(2)]
    else:
        state["out"] = [torch.empty_like(q)]
    return state


# ---- the plain form -------------------------------------------------------------
def _blocks(x):
    """(bytes of two codes [n, width / 2], f16 scales [n, width / 32]) of rows x [n, width]."""
    n, width = x.shape
    b = x.view(n, width // 32, 32)
    peak = b.gather(2, b.abs().argmax(2, keepdim=True))
    d = (peak / -8).half()
    f = d.float()
    r = torch.where(f != 0, 1 / f, 0.0)
    c = (b * r + 8.5).clamp(0, 15).to(torch.uint8).view(n, width // 2, 2)
    return c[..., 0] | (c[..., 1] << 4), d.view(n, width // 32)


def _values(blocks):
    """The f32 rows [n, width] that blocks stand for."""
    c, d = blocks
    n, half = c.shape
    x = torch.stack((c & 15, c >> 4), 2).view(n, d.shape[1], 32).float()
    return ((x - 8) * d.float()[..., None]).view(n, 2 * half)


def _heads(x, G, d):
    """Rows [n, G * d] as [G, n, d]."""
    return x.view(x.shape[0], G, d).transpose(0, 1).contiguous()


def _plain(state):
    case = state["case"]
    H, G, d = case["H"], case["G"], case["d"]
    if case["op"] == "write":
        blocks = [_blocks(x) for x in state["new"]]
        if state["old"] is not None:
            blocks = [tuple(torch.cat(p) for p in zip(o, b)) for o, b in zip(state["old"], blocks)]
        return {"k": _values(blocks[0]), "v": _values(blocks[1])}
    k, v = (_values(b) for b in state["old"])
    if case["op"] == "read":
        return {"k": k, "v": v}
    q = state["q"]
    T, n, rep = q.shape[0], k.shape[0], H // G
    rows = q.view(T, G, rep, d).transpose(0, 1).reshape(G, T * rep, d)
    s = torch.matmul(rows, _heads(k, G, d).transpose(1, 2).contiguous()) * (1 / math.sqrt(d))
    if T > 1:
        seen = torch.arange(n, device="cuda")[None] <= n - T + torch.arange(T, device="cuda")[:, None]
        s = torch.where(seen.repeat_interleave(rep, 0), s, -math.inf)
    p = (s - s.amax(2, keepdim=True)).exp()
    o = torch.matmul(p, _heads(v, G, d)) / p.sum(2, keepdim=True)
    return o.view(G, T, rep, d).transpose(0, 1).reshape(T, H * d)


# ---- the framework's calls --------------------------------------------------------
def _calls(state):
    case, cache = state["case"], state["cache"]
    out = [_Buffer(t) for t in state["out"]]
    if case["op"] == "write":
        k, v = (_Buffer(x) for x in state["new"])
        cache.truncate(0, case["base"])
        cache.append(0, k, v, case["T"])
        cache.dequant_into(0, case["base"] + case["T"], out[0], out[1])
    elif case["op"] == "read":
        cache.dequant_into(0, case["ctx"], out[0], out[1])
    elif case["op"] == "decode":
        cache.attention_decode(0, _Buffer(state["q"]), out[0], case["H"], case["ctx"], 1 / math.sqrt(case["d"]))
    else:
        cache.attention_chunk(0, _Buffer(state["q"]), out[0], case["H"], case["T"], case["ctx"], 1 / math.sqrt(case["d"]))
    if state["q"] is None:
        return {"k": state["out"][0], "v": state["out"][1]}
    return state["out"][0]


def run(state):
    """One pass.  The framework's calls are queued on its context's stream: what they return is
    there after Context.sync() or torch.cuda.synchronize()."""
    return _calls(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    H, G, d = case["H"], case["G"], case["d"]
    element = 18 / 32
    if case["op"] == "write":
        new, n = 2 * case["T"] * G * d, 2 * (case["base"] + case["T"]) * G * d
        old = n - new
        return {"bytes": new * (4 + element) + old * element + n * 4, "flops": 8 * new + 2 * n}
    n = 2 * case["ctx"] * G * d
    if case["op"] == "read":
        return {"bytes": n * (element + 4), "flops": 2 * n}
    T, ctx = case.get("T", 1), case["ctx"]
    seen = T * (ctx - T) + T * (T + 1) // 2
    return {"bytes": n * element + 2 * T * H * d * 4, "flops": 4 * H * d * seen}


# ---- the same in 64 bits -----------------------------------------------------------
def _stored64(x):
    """What the cache holds of rows x, by the definition above: every rounding that it names made one by one."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[0], 8192):
        w = x[at:at + 8192].double()
        b = w.reshape(-1, 32)
        top, low = b.max(1), b.min(1)
        up = (top.values > -low.values) | ((top.values == -low.values) & (top.indices < low.indices))
        peak = torch.where(up, top.values, low.values)
        scale = (peak * -0.125).float().to(torch.float16).double()[:, None]
        inverse = torch.where(scale == 0, torch.zeros_like(scale), (1 / scale).float().double())
        code = ((b * inverse).float().double() + 8.5).float().double().trunc().clamp(0, 15)
        out[at:at + 8192] = ((code - 8) * scale).reshape(w.shape)
    return out


def exact(case, seed):
    H, G, d = case["H"], case["G"], case["d"]
    old, new, q = _inputs(case, seed)
    if q is None:
        parts = [p for p in (old, new) if p is not None]
        return {"k": torch.cat([_stored64(p[0]) for p in parts]), "v": torch.cat([_stored64(p[1]) for p in parts])}
    k, v = _stored64(old[0]), _stored64(old[1])
    T, n = q.shape[0], k.shape[0]
    out = torch.empty(T, H * d, dtype=torch.float64, device="cuda")
    rows, keys = torch.arange(T, device="cuda"), torch.arange(n, device="cuda")
    hidden = keys[None, :] > (rows + n - T)[:, None]
    for h in range(H):
        g = h // (H // G)
        kh, vh = k[:, g * d:(g + 1) * d], v[:, g * d:(g + 1) * d]
        s = (q[:, h * d:(h + 1) * d].double() @ kh.t()) / d ** 0.5
        p = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
        out[:, h * d:(h + 1) * d] = p @ vh
    return out
