"""The attention side of a decoder layer on one MI355X: head norms and rotation, the quantized cache, attention.

``listed()`` holds the fixed cases, ``draw(rng)`` more of the same kinds over the whole range of sizes. A case is a
dict of plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass: with ``own`` false
in plain torch, with ``own`` true through the public entry points of ``brimkern_amd.Context``; ``exact`` computes the
same outputs in 64 bits. Kinds:

``rope``     queries and keys of a step: RMS norm of every head, then the rotation by the row's position
``append``   the same with the keys and values of the step quantized into their cache slots, and read back from there
``write``    keys and values quantized into the cache as they are, and read back
``attn``     attention of the step's rows over the quantized cache (one row a sequence: decoding; many: prefill)
``prefix``   the same where all sequences share a prefix that lies in the cache once

A cache is ``.brik`` q8 or q4 planes of ``[pages, kv heads, page, head dim]`` values for keys and for values; a
sequence's tokens lie in the pages of its row of the table, in order. The rows of a step are the last tokens of their
sequences: row t of the n rows of a sequence of L tokens has position L - n + t and sees the keys up to its own
position (``window``: only that many of them, its own included). A row that sees no key gives zeros.

The library's context has a stream of its own, which does not wait for torch's and which torch's does not wait for. So with
``own`` true ``prepare`` returns when its inputs are there; what ``run`` returns is there after ``context().sync()`` (or
``torch.cuda.synchronize()``, which waits for every stream), and a state is kept until then.
"""
import math

import torch

DEV = "cuda:0"
own = False
EPS = 1e-6

_context = None


def context():
    """The one library context of the process (a program keeps it for its lifetime)."""
    global _context
    if _context is None:
        from brimkern_amd import Context
        _context = Context(0)
    return _context


# B sequences, up to L tokens each (ragged: from 1 to L, one of them L), n rows each in this step (ragged: 1 to n);
# H query heads, KV kv heads, D values per head, P tokens per page
_Q4B = {"H": 32, "KV": 8, "D": 128}           # the heads of Qwen3-4B
_SMALL = {"H": 14, "KV": 2, "D": 64}          # the heads of a 0.5B model


def listed():
    return [
        # one token of one sequence: the norms and rotations of its 40 heads
        {"name": "rope_decode_1", "kind": "rope", **_step(1, 700, 1), **_Q4B, **_rot(128)},
        # a prompt of 2048 tokens
        {"name": "rope_prefill_2048", "kind": "rope", **_step(1, 2048, 2048), **_Q4B, **_rot(128)},
        # 64 sequences decoded together: their new keys and values into a q8 cache
        {"name": "append_q8_decode_64", "kind": "append", "fmt": "q8", **_step(64, 4096, 1, ragged=True), **_Q4B, **_rot(128)},
        # three prompts of odd lengths into a q4 cache, a small model
        {"name": "append_q4_prefill_3x777", "kind": "append", "fmt": "q4", **_step(3, 777, 777, ragged=True), **_SMALL,
         **_rot(64, norm=False)},
        # keys and values that another program computed: 4096 tokens into a q8 cache and back
        {"name": "write_q8_4096", "kind": "write", "fmt": "q8", **_step(1, 4096, 4096), **_Q4B},
        # one sequence, one token: the call that a single user waits for
        {"name": "decode_q8_1x4095", "kind": "attn", "fmt": "q8", **_step(1, 4095, 1), **_Q4B, **_mask()},
        # a serving batch of sequences of all lengths
        {"name": "decode_q4_32x8192", "kind": "attn", "fmt": "q4", **_step(32, 8192, 1, ragged=True), **_Q4B, **_mask()},
        # a very long sequence
        {"name": "decode_q8_1x131072", "kind": "attn", "fmt": "q8", **_step(1, 131072, 1), **_Q4B, **_mask()},
        # a whole prompt: the largest
        {"name": "prefill_q8_4096", "kind": "attn", "fmt": "q8", **_step(1, 4096, 4096), **_Q4B, **_mask()},
        # pieces of five prompts on top of what is there, with a sliding window and capped scores
        {"name": "prefill_q4_5x333_window", "kind": "attn", "fmt": "q4", **_step(5, 5000, 333, ragged=True), **_SMALL,
         **_mask(window=1024, softcap=50.0)},
        # 64 sequences decoded behind one system prompt
        {"name": "prefix_q8_64x8192", "kind": "prefix", "fmt": "q8", **_step(64, 8192 + 300, 1, ragged=True), **_Q4B, **_mask(),
         "prefix": 8192},
        # nine drafts of three tokens behind a prefix that ends inside a page
        {"name": "prefix_q4_9x3x2001", "kind": "prefix", "fmt": "q4", **_step(9, 2001 + 77, 3, ragged=True), **_Q4B, **_mask(),
         "prefix": 2001},
    ]


def _step(B, L, n, ragged=False, P=64):
    return {"B": B, "L": L, "n": n, "ragged": ragged, "P": P}


def _rot(rot, norm=True, interleaved=False, one_plus=False):
    return {"rot": rot, "norm": norm, "interleaved": interleaved, "one_plus": one_plus, "base": 1e6}


def _mask(window=0, softcap=0.0):
    return {"window": window, "softcap": softcap}


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


LARGEST = 32 * 4096 * 4096 * 128              # of the largest listed case: query heads x rows x keys x head dim


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "write", "attn", "attn", "attn", "attn", "prefix", "prefix"])
    D = rng.choice([64, 96, 128, 128, 192, 256])
    KV = rng.choice([1, 2, 4, 8])
    H = KV * rng.choice([1, 2, 3, 4, 5, 7, 8])
    c = {"kind": kind, "fmt": rng.choice(["q8", "q4"]), "H": H, "KV": KV, "D": D}
    P, ragged = rng.choice([16, 32, 64, 128, 256]), rng.random() < 0.6
    if kind in ("rope", "append", "write"):
        B = _log(rng, 1, 64)
        n = 1 if rng.random() < 0.4 else _log(rng, 1, 4096 // B)
        c.update(_step(B, n + _log(rng, 1, 4096), n, ragged, P))
        if kind != "write":
            c.update(_rot(rng.choice([D, D, D // 2]), rng.random() < 0.7, rng.random() < 0.3, rng.random() < 0.3))
        if kind == "rope":
            del c["fmt"]
        return c
    prefix = _log(rng, 33, 16384) if kind == "prefix" else 0
    B = _log(rng, 1, 64)
    L = _log(rng, 1, 500 if prefix else 131072 // B)
    n = min(L, 1 if rng.random() < 0.5 else _log(rng, 1, 2048))
    n = max(1, min(n, LARGEST // 2 // (H * D * (L + prefix)) // B))
    c.update(_step(B, prefix + L, n, ragged, P),
             **_mask(_log(rng, 16, 4096) if rng.random() < 0.2 else 0, 50.0 if rng.random() < 0.2 else 0.0))
    if prefix:
        c["prefix"] = prefix
    return c


# ---- inputs --------------------------------------------------------------------------------------


def _plan(c):
    """Rows and lengths of the sequences, by the case alone: (rows n_b, tokens L_b, own tokens behind the prefix)."""
    B, L, n, prefix = c["B"], c["L"], c["n"], c.get("prefix", 0)
    part = [1.0 if not c["ragged"] or b == B // 2 else (b + 1) * 0.6180339887498949 % 1.0 for b in range(B)]
    rows = [max(1, round(n * p)) for p in part]
    lens = [max(r, round((L - prefix) * p)) + prefix for r, p in zip(rows, part)]
    return rows, lens, [x - prefix for x in lens]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _heads(g, T, heads, D):
    """Rows of heads [T, heads, D]: normal, with a log-normal gain per channel."""
    gain = torch.exp(0.4 * torch.randn(heads, D, generator=g, device=DEV))
    return torch.randn(T, heads, D, generator=g, device=DEV) * gain


def _half_bits(v):
    """binary16 bits of f64 values as the ``.brik`` encoders round them: to f32, then the mantissa half up, below the
    normal range 0, above it 65504."""
    x = v.to(torch.float32).view(torch.int32)
    e = ((x >> 23) & 255) - 112
    body = (e << 10) + ((x >> 13) & 1023) + ((x >> 12) & 1)
    body = torch.where(e <= 0, 0, torch.where(e >= 31, 0x7BFF, body))
    return (((x >> 16) & 0x8000) | body).to(torch.int16)


def _f64(bits):
    return bits.view(torch.float16).to(torch.float64)


def encode(fmt, x):
    """Planes of f32 values in groups of 32 along the last axis: (codes, scales) or (nibbles, scales, mins)."""
    gr = x.to(torch.float64).unflatten(-1, (-1, 32))
    levels = torch.tensor([127.0 if fmt == "q8" else 15.0], dtype=torch.float64, device=DEV)     # (x / 127.0 would multiply)
    if fmt == "q8":
        sc = gr.abs().amax(-1) / levels
        lo, hi, mn = -127, 127, None
    else:
        mn = _half_bits(gr.amin(-1))
        sc = (gr.amax(-1) - gr.amin(-1)) / levels
        lo, hi = 0, 15
    sc = _half_bits(torch.where(sc == 0, 1e-8, sc))
    s = _f64(sc)
    s = torch.where(s == 0, 1e-8, s)[..., None]
    q = torch.floor((gr if mn is None else gr - _f64(mn)[..., None]) / s + 0.5).clamp_(lo, hi).flatten(-2)
    if fmt == "q8":
        return q.to(torch.int8), sc
    q = q.to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), sc, mn


def decode(fmt, planes, dtype=torch.float32):
    """The values of planes whose last axis is one head, [..., D]."""
    if fmt == "q8":
        q, (sc, mn) = planes[0], (planes[1], None)
    else:
        q, (sc, mn) = torch.stack((planes[0] & 15, planes[0] >> 4), -1).flatten(-2), planes[1:]
    v = q.unflatten(-1, (-1, 32)).to(dtype) * sc.view(torch.float16).to(dtype)[..., None]
    return (v if mn is None else v + mn.view(torch.float16).to(dtype)[..., None]).flatten(-2)


def _empty_planes(fmt, pages, c):
    KV, P, D = c["KV"], c["P"], c["D"]
    code = torch.zeros(pages, KV, P, D if fmt == "q8" else D // 2, dtype=torch.int8 if fmt == "q8" else torch.uint8, device=DEV)
    half = [torch.zeros(pages, KV, P, D // 32, dtype=torch.int16, device=DEV) for _ in range(1 if fmt == "q8" else 2)]
    return [code, *half]


def _inputs(c, seed):
    """The tensors of a case, from the seed alone."""
    g, kind, P, D = _gen(seed), c["kind"], c["P"], c["D"]
    rows, lens, mine = _plan(c)
    T, B, prefix = sum(rows), c["B"], c.get("prefix", 0)
    off = [0]
    for r in rows:
        off.append(off[-1] + r)
    s = {"kv_len": _ints(lens), "row_off": _ints(off)}
    # the pages: drawn from a pool a little larger than needed, in no order
    cols, pre = max(-(-x // P) for x in mine), -(-prefix // P)
    need = sum(-(-x // P) for x in mine) + pre
    pages = need + 1 + need // 8
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table, at = [], pre
    for x in mine:
        k = -(-x // P)
        table.append(list(range(at, at + k)) + [at + k - 1] * (cols - k))
        at += k
    s["table"], s["prefix_table"] = order[_ints(table).long()].contiguous(), order[:pre].contiguous()
    if kind in ("rope", "append", "write"):
        s["k"], s["v"] = _heads(g, T, c["KV"], D), _heads(g, T, c["KV"], D)
        if kind != "write":
            s["q"] = _heads(g, T, c["H"], D)
            s["freq"] = (1.0 / c["base"] ** (torch.arange(0, c["rot"], 2, dtype=torch.float64, device=DEV) / c["rot"])).to(torch.float32)
            for w in ("q_norm", "k_norm"):
                s[w] = (0.0 if c["one_plus"] else 1.0) + 0.1 * torch.randn(D, generator=g, device=DEV)
        if kind != "rope":
            s["kc"], s["vc"] = _empty_planes(c["fmt"], pages, c), _empty_planes(c["fmt"], pages, c)
        return s
    s["q"] = _heads(g, T, c["H"], D)
    for n in ("kc", "vc"):
        s[n] = list(encode(c["fmt"], _heads(g, pages * P, c["KV"], D).view(pages, P, c["KV"], D).transpose(1, 2).contiguous()))
    return s


def _at(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _handles(s):
    """What a program makes once of its buffers: the cache, the step's batch and the arguments of its calls."""
    ctx, c = context(), s["case"]
    kind, D = c["kind"], c["D"]
    h = {"batch": ctx.kv_batch(seqs=c["B"], rows=s["T"], row_off=_at(s["row_off"]), kv_len=_at(s["kv_len"]), table=_at(s["table"]),
                               table_cols=s["table"].shape[1], max_len=c["L"], max_rows=c["n"], prefix_table=_at(s["prefix_table"]),
                               prefix_len=c.get("prefix", 0))}
    if kind != "rope":
        h["cache"] = ctx.kv_cache(c["fmt"], c["KV"], D, c["P"], s["kc"][0].shape[0], [_at(p) for p in s["kc"]], [_at(p) for p in s["vc"]])
    if kind in ("attn", "prefix"):
        h["args"] = ctx.attn_args(q=_at(s["q"]), out=_at(s["out"]), heads=c["H"], scale=1 / math.sqrt(D), window=c["window"],
                                  softcap=c["softcap"])
    elif kind == "write":
        h["rows"] = ctx.qkv_rows(head_dim=D, kv_heads=c["KV"], k=_at(s["k"]), v=_at(s["v"]))
    else:
        norm = {"q_norm": _at(s["q_norm"]), "k_norm": _at(s["k_norm"])} if c["norm"] else {}
        h["rows"] = ctx.qkv_rows(head_dim=D, heads=c["H"], kv_heads=c["KV"], q=_at(s["q"]), k=_at(s["k"]), v=_at(s["v"]),
                                 q_out=_at(s["q_out"]), k_out=_at(s["k_out"]) if kind == "rope" else None, eps=EPS, inv_freq=_at(s["freq"]),
                                 rot_dim=c["rot"], interleaved=c["interleaved"], one_plus=c["one_plus"], **norm)
    return h


def prepare(case, seed):
    s = {**_inputs(case, seed), "case": dict(case)}
    T, c = sum(_plan(case)[0]), case
    s["T"] = T
    if c["kind"] in ("attn", "prefix"):
        s["out"] = torch.zeros(T, c["H"], c["D"], device=DEV)
    else:
        s["k_out"], s["v_out"] = (torch.zeros(T, c["KV"], c["D"], device=DEV) for _ in range(2))
        s["q_out"] = torch.zeros(T, c["H"], c["D"], device=DEV) if c["kind"] != "write" else None
    if own:
        s["h"] = _handles(s)
        torch.cuda.synchronize()                         # the library's stream does not wait for torch's
    return s


# ---- one pass ------------------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        ctx, h = context(), s["h"]
        if kind == "rope":
            ctx.qk_norm_rope(h["batch"], h["rows"])
            return {"q": s["q_out"], "k": s["k_out"]}
        if kind in ("attn", "prefix"):
            ctx.attention(h["cache"], h["batch"], h["args"])
            return s["out"]
        ctx.kv_write(h["cache"], h["batch"], h["rows"])
        ctx.kv_read(h["cache"], h["batch"], _at(s["k_out"]), _at(s["v_out"]))
        return {"k": s["k_out"], "v": s["v_out"], **({"q": s["q_out"]} if kind == "append" else {})}
    if kind == "rope":
        return {"q": _norm_rope(s, s["q"], s["q_norm"]), "k": _norm_rope(s, s["k"], s["k_norm"])}
    if kind in ("attn", "prefix"):
        return _attention(s)
    fmt, got = s["case"]["fmt"], {}
    page, slot = _slots(s)
    k = s["k"] if kind == "write" else _norm_rope(s, s["k"], s["k_norm"])
    kc, vc = encode(fmt, k), encode(fmt, s["v"])
    got["k"] = _stored(fmt, s["kc"], kc, page, slot)
    got["v"] = _stored(fmt, s["vc"], vc, page, slot)
    if kind == "append":
        got["q"] = _norm_rope(s, s["q"], s["q_norm"])
    return got


def _rows_of(s):
    """The sequence and the position of every row."""
    off, n = s["row_off"].long(), s["T"]
    row = torch.arange(n, device=DEV)
    seq = torch.searchsorted(off[1:], row, right=True)
    return seq, s["kv_len"].long()[seq] - off[seq + 1] + row


def _norm_rope(s, x, w):
    """Every head of x [T, heads, D] normed by its root mean square, then rotated: in 64 bits, rounded once."""
    c, y = s["case"], x.to(torch.float64)
    if c["norm"]:
        gain = w.to(torch.float64) + (1.0 if c["one_plus"] else 0.0)
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * gain
    angle = (_rows_of(s)[1].to(torch.float64)[:, None] * s["freq"].to(torch.float64))[:, None, :]
    cos, sin, rot = torch.cos(angle), torch.sin(angle), c["rot"]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if c["interleaved"] else (y[..., : rot // 2], y[..., rot // 2:rot])
    pair = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(pair, -1).flatten(-2) if c["interleaved"] else torch.cat(pair, -1)
    return torch.cat((turned, y[..., rot:]), -1).to(torch.float32)


def _slots(s):
    seq, pos = _rows_of(s)
    P = s["case"]["P"]
    return s["table"].long()[seq, pos // P], pos % P


def _stored(fmt, cache, planes, page, slot):
    """The rows' planes put into the cache, and what the cache then holds there."""
    for dst, src in zip(cache, planes):
        dst[page, :, slot] = src
    return decode(fmt, [p[page, :, slot] for p in cache])


def _keys(s, name, table):
    """The values in the pages of ``table`` [..., cols]: [..., kv heads, cols * P, D]."""
    c = s["case"]
    v = decode(c["fmt"], [p[table.long()] for p in s[name]])
    return v.movedim(-3, -4).flatten(-3, -2)


def _attention(s):
    c = s["case"]
    B, KV, D, G, prefix = c["B"], c["KV"], c["D"], c["H"] // c["KV"], c.get("prefix", 0)
    off, lens = s["row_off"].long(), s["kv_len"].long()
    n = c["n"]
    rows = off[:-1, None] + torch.arange(n, device=DEV)
    real = rows < off[1:, None]
    q = s["q"][torch.where(real, rows, 0)].view(B, n, KV, G, D).permute(0, 2, 3, 1, 4)          # [B, KV, G, n, D]
    pos = (lens - (off[1:] - off[:-1]))[:, None] + torch.arange(n, device=DEV)                  # [B, n]
    k, v = _keys(s, "kc", s["table"]), _keys(s, "vc", s["table"])
    x = _scores(c, (q.reshape(B, KV, G * n, D) @ k.transpose(-1, -2)).view(B, KV, G, n, -1), pos, prefix, lens)
    if prefix:
        kp, vp = (_keys(s, w, s["prefix_table"])[:, :prefix] for w in ("kc", "vc"))
        q1 = q.permute(1, 0, 2, 3, 4).reshape(KV, B * G * n, D)
        xp = (q1 @ kp.transpose(-1, -2)).view(KV, B, G, n, prefix).transpose(0, 1)
        x = torch.cat((_scores(c, xp, pos, 0, lens), x), -1)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = (p[..., prefix:].reshape(B, KV, G * n, -1) @ v).view(B, KV, G, n, D)
    if prefix:
        o = o + (p[..., :prefix].transpose(0, 1).reshape(KV, B * G * n, prefix) @ vp).view(KV, B, G, n, D).transpose(0, 1)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, KV * G, D)[real]


def _scores(c, x, pos, first, lens):
    """Scaled and capped scores [B, KV, G, n, keys] of the keys at positions ``first`` and on, masked."""
    x = x * (1 / math.sqrt(c["D"]))
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    key = first + torch.arange(x.shape[-1], device=DEV)
    seen = (key <= pos[..., None]) & (key < lens[:, None, None])
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    return torch.where(seen[:, None, None], x, -math.inf)


# ---- what a pass cannot do without ---------------------------------------------------------------


def _cached(c, tokens):
    """Bytes of ``tokens`` tokens in the cache, keys and values."""
    n = 2 * tokens * c["KV"] * c["D"]
    return n + n // 16 if c["fmt"] == "q8" else n // 2 + n // 8


def work(case):
    c, kind = case, case["kind"]
    rows, lens, mine = _plan(c)
    T, D, H, KV, prefix = sum(rows), c["D"], c["H"], c["KV"], c.get("prefix", 0)
    if kind == "rope":
        return {"bytes": 8 * T * (H + KV) * D, "flops": 7 * T * (H + KV) * D}
    if kind in ("append", "write"):
        heads = 2 * KV if kind == "write" else H + 2 * KV
        back = 8 * T * KV * D                              # keys and values read back
        return {"bytes": 4 * T * heads * D + (4 * T * H * D if kind == "append" else 0) + 2 * _cached(c, T) + back,
                "flops": 7 * T * heads * D}
    pairs, read, shared = 0, 0, 0
    for r, n, m in zip(rows, lens, mine):
        w = c["window"] or n
        pairs += sum(min(n - r + t + 1, w) for t in range(r))
        read += max(0, min(m, w + r - 1))
        shared = max(shared, min(prefix, max(0, w + r - 1 - m)))
    return {"bytes": _cached(c, read + shared) + 8 * T * H * D, "flops": 4 * pairs * H * D}


# ---- the same in 64 bits -------------------------------------------------------------------------


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    kind, rows, lens = c["kind"], *_plan(case)[:2]
    if kind in ("attn", "prefix"):
        if 4 * max(rows) * max(lens) * c["H"] * 8 > 40e9:
            return None
        return _exact_attention(c, s, rows, lens)
    fmt, f64 = c.get("fmt"), torch.float64

    def turned(x, w):
        """One pair of every head at a time, as a product of complex numbers."""
        y = x.to(f64)
        if c["norm"]:
            y = y * torch.rsqrt(y.square().sum(-1, keepdim=True) / c["D"] + EPS) * (w.to(f64) + int(c["one_plus"]))
        at = torch.cat([torch.arange(n - r, n, device=DEV) for r, n in zip(rows, lens)]).to(f64)
        half = c["rot"] // 2
        i = torch.arange(half, device=DEV)
        a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
        angle = torch.outer(at, s["freq"].to(f64))
        z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        out = y.clone()
        out[..., a], out[..., b] = z.real, z.imag
        return out

    def half(v):
        """The binary16 value of f64 values by arithmetic: multiples of 2^-10 of the power of two below, half up."""
        v = v.to(torch.float32).to(f64)
        step = torch.ldexp(torch.ones_like(v), torch.frexp(v)[1] - 11)
        near = torch.floor(v.abs() / step + 0.5) * step * torch.sign(v)
        return torch.where(v.abs() < 2.0**-14, 0.0, near)

    def held(x):
        """The values that a cache of this format holds for the f32 rows x."""
        x = x.to(torch.float32).to(f64).unflatten(-1, (-1, 32))
        count = torch.full_like(x[..., :1], 127 if fmt == "q8" else 15)
        if fmt == "q8":
            step = half(x.abs().max(-1, keepdim=True)[0] / count)
            return (step * torch.floor(x / step + 0.5).clamp(-127, 127)).flatten(-2)
        low, high = x.min(-1, keepdim=True)[0], x.max(-1, keepdim=True)[0]
        step, least = half((high - low) / count), half(low)
        return (step * torch.floor((x - least) / step + 0.5).clamp(0, 15) + least).flatten(-2)

    if kind == "rope":
        return {"q": turned(s["q"], s["q_norm"]), "k": turned(s["k"], s["k_norm"])}
    k = s["k"] if kind == "write" else turned(s["k"], s["k_norm"])
    got = {"k": held(k), "v": held(s["v"])}
    if kind == "append":
        got["q"] = turned(s["q"], s["q_norm"])
    return got


def _exact_attention(c, s, rows, lens):
    """Sequence by sequence, over the keys of its own tokens in order."""
    f64, KV, D, G, P, prefix = torch.float64, c["KV"], c["D"], c["H"] // c["KV"], c["P"], c.get("prefix", 0)
    outs, at = [], 0
    for b, (r, n) in enumerate(zip(rows, lens)):
        token = torch.arange(n, device=DEV)
        own_token = (token - prefix).clamp_min(0)
        page = s["table"][b].long()[own_token // P]
        slot = torch.where(token < prefix, token, own_token) % P
        if prefix:
            page = torch.where(token < prefix, s["prefix_table"].long()[token.clamp_max(prefix - 1) // P], page)
        k, v = (decode(c["fmt"], [p[page, :, slot] for p in s[w]], f64).transpose(0, 1).contiguous() for w in ("kc", "vc"))
        q = s["q"][at:at + r].to(f64).view(r, KV, G, D).permute(1, 2, 0, 3).reshape(KV, G * r, D)
        x = torch.bmm(q, k.transpose(1, 2).contiguous()).view(KV, G, r, n) / math.sqrt(D)
        if c["softcap"]:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        back = torch.arange(n - r, n, device=DEV)[:, None] - token            # how far behind the row the key lies
        hidden = (back < 0) | (back >= (c["window"] or n + 1))
        p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
        outs.append(torch.bmm(p.view(KV, G * r, n), v).view(KV, G, r, D).permute(2, 0, 1, 3).reshape(r, KV * G, D))
        at += r
    return torch.cat(outs)
