"""The 4-bit key/value cache and the attention that reads it, as measurable
cases: storing K and V rows (and reading them back), reading stored rows back,
attention of one token, of a batch of sequences and of a prompt's rows.

A cache is a pool of pages.  A page holds `page` tokens of every kv head; the
page table of a sequence lists its pages in order.  32 elements of a head's row
share one fp16 scale:

    a = max |x|,  s = min(fp16(a / 7), 9352),  q = sign(x) min(7, floor(|x| / s + 1/2))

and the stored nibble is q + 8.  Per page and kv head the bytes are the K
nibbles, the V nibbles and the scales (see _views below for their order).

`own` selects who computes: the plain torch form, or madi_amd.kv4.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
QMAX = 7
SCALE_MAX = 9352.0  # the largest fp16 s with 7 s finite in fp16


# ---------------------------------------------------------------- the cases
def _case(name, op, dtype, nh, nkv, d, page, b, len_lo, len_hi, rows_lo, rows_hi, causal=True, window=0):
    return dict(name=name, op=op, dtype=dtype, nh=nh, nkv=nkv, d=d, page=page, b=b, len_lo=len_lo,
                len_hi=len_hi, rows_lo=rows_lo, rows_hi=rows_hi, causal=causal, window=window)


def listed():
    return [
        # the batched decoder's cache write: one new f32 row for each of 8 slots
        # of the Whisper decoder (20 heads of 64, up to 448 positions)
        _case("store_step_8", "store", "f32", 20, 20, 64, 64, 8, 57, 430, 1, 1),
        # a serving step with new prompts of odd lengths beside running sequences
        _case("store_ragged_24", "store", "f16", 32, 8, 128, 16, 24, 64, 2500, 1, 511),
        # long prompts stored whole
        _case("store_prompt_4x4096", "store", "f16", 32, 8, 128, 64, 4, 4096, 4096, 4096, 4096),
        # a window's cross-attention rows read back (1500 frames, 20 heads of 64)
        _case("load_window_1500", "load", "f32", 20, 20, 64, 64, 1, 1500, 1500, 1500, 1500),
        # caches of long sequences read back whole, to hand them to other code
        _case("load_long_8x16384", "load", "f16", 32, 8, 128, 32, 8, 16384, 16384, 16384, 16384),
        # one token of one sequence, the decoder's self-attention: latency
        _case("attn_step_1", "attn", "f32", 20, 20, 64, 64, 1, 213, 213, 1, 1),
        # its cross-attention, 8 slots over a window's 1500 encoder rows
        _case("attn_cross_8x1500", "attn", "f32", 20, 20, 64, 64, 8, 1500, 1500, 1, 1, causal=False),
        # a serving batch: one token each, lengths from 1 to 8000, grouped heads
        _case("attn_ragged_48", "attn", "f16", 32, 8, 128, 16, 48, 1, 8000, 1, 1),
        # one long document
        _case("attn_long_131072", "attn", "f16", 32, 8, 128, 256, 1, 131072, 131072, 1, 1),
        # a full batch of long sequences: 1.2 GB of cache a pass
        _case("attn_batch_128x8192", "attn", "f16", 32, 8, 128, 64, 128, 8192, 8192, 1, 1),
        # the Whisper decoder's prompts (at most 224 tokens), four slots, f32
        _case("attn_prompt_4x224", "attn", "f32", 20, 20, 64, 64, 4, 31, 230, 17, 224),
        # a prompt's next chunk over the cache of what came before
        _case("attn_prompt_2048", "attn", "f16", 32, 8, 128, 64, 1, 16384, 16384, 2048, 2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "load", "attn", "attn", "attn"])
    dtype = rng.choice(["f16", "f32"])
    d = rng.choice([64, 64, 96, 128, 128, 256])
    nkv = rng.choice([1, 2, 4, 8, 8, 20])
    nh = nkv * (rng.choice([1, 2, 4, 5, 8, 16]) if nkv <= 8 else 1)
    page = rng.choice([16, 32, 64, 128, 256])
    if op != "attn":
        b = _log(rng, 1, 32)
        hi = _log(rng, 1, max(1, (64 << 20) // (b * nkv * d)))
        lo = rng.choice([1, max(1, hi // 3), hi])
        rows = rng.choice([1, hi, max(1, hi // 2)])
        return _case("", op, dtype, nh, nkv, d, page, b, lo, hi, min(1 + rows // 5, rows), rows)
    if rng.random() < 0.65:  # one token, or a few (a draft's tokens), per sequence
        b = _log(rng, 1, 128)
        hi = _log(rng, 1, min(131072, max(64, (512 << 20) // (b * nkv * d))))
        lo = rng.choice([1, max(1, hi // 4), hi])
        rows = rng.choice([1, 1, 1, 2, 5])
        causal = rng.random() < 0.8
        window = _log(rng, 16, 4096) if causal and rng.random() < 0.25 else 0
        return _case("", op, dtype, nh, nkv, d, page, b, lo, hi, 1, rows, causal, window)
    b = rng.choice([1, 1, 2, 4, 7])
    rows = _log(rng, 8, 2048 // b)
    # at most the listed prompt's products
    hi = max(rows, _log(rng, rows, max(rows + 1, min(16384, (1 << 36) // (b * rows * nh * d)))))
    causal = rng.random() < 0.8
    window = _log(rng, 64, 4096) if causal and rng.random() < 0.25 else 0
    return _case("", op, dtype, nh, nkv, d, page, b, rng.choice([hi, max(1, hi // 2)]), hi,
                 rng.choice([rows, 1 + rows // 3]), rows, causal, window)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced in their logarithm, in an
    order that is not sorted."""
    out = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]
    if n == 1:
        out = [hi]
    step = next(s for s in (5, 7, 11, 13) if math.gcd(s, n) == 1)
    return [out[(i * step) % n] for i in range(n)]


def _shape(case):
    lens = _spread(case["len_lo"], case["len_hi"], case["b"])
    rows = _spread(case["rows_lo"], case["rows_hi"], case["b"])
    return lens, [min(r, n) for r, n in zip(rows, lens)]


def _visible(case, n, rows):
    """(row, key) pairs that are not masked, and the keys some row sees."""
    if not case["causal"]:
        return rows * n, n
    w = case["window"] or n
    pairs = sum(min(p + 1, w) for p in range(n - rows, n))
    return pairs, min(n, w + rows - 1)


def work(case):
    lens, rows = _shape(case)
    esize = 4 if case["dtype"] == "f32" else 2
    width = case["nkv"] * case["d"]
    token = 2 * width // 2 + 2 * width // BLOCK * 2  # nibbles and scales of K and V
    m = sum(rows)
    if case["op"] == "store":  # rows in, rows held, rows back out
        return dict(bytes=m * (2 * width * esize * 2 + token), flops=m * 2 * width * 6)
    if case["op"] == "load":
        return dict(bytes=m * (2 * width * esize + token), flops=m * 2 * width)
    seen = [_visible(case, n, r) for n, r in zip(lens, rows)]
    return dict(bytes=sum(k for _, k in seen) * token + 2 * m * case["nh"] * case["d"] * esize,
                flops=sum(p for p, _ in seen) * 4 * case["nh"] * case["d"])


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(gen, n, heads, d, dtype, outliers):
    """K or V rows: N(0, 1), and for K a few channels of a head much larger, as
    keys have them."""
    x = torch.randn(n, heads, d, generator=gen, device="cuda")
    if outliers:
        big = torch.rand(heads, d, generator=gen, device="cuda") < 0.04
        x *= torch.where(big, 5.0, 1.0)
    return x.to(dtype)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _make(case, seed):
    """Everything made from the seed: per sequence the rows its cache holds in
    natural order (codes and scales), the new rows or the queries."""
    gen = _generator(seed)
    lens, rows = _shape(case)
    nkv, d, dt = case["nkv"], case["d"], _dtype(case)
    m = sum(rows)
    made = dict(lens=lens, rows=rows)
    if case["op"] == "store":
        kv = torch.empty(m, 2, nkv, d, dtype=dt, device="cuda")
        kv[:, 0] = _rows(gen, m, nkv, d, dt, True)
        kv[:, 1] = _rows(gen, m, nkv, d, dt, False)
        made["kv"] = kv
    else:
        made["held"] = [(_held(_rows(gen, n, nkv, d, torch.float16, True)),
                         _held(_rows(gen, n, nkv, d, torch.float16, False))) for n in lens]
        if case["op"] == "attn":
            made["q"] = torch.randn(m, case["nh"], d, generator=gen, device="cuda").to(dt)
    made["gen"] = gen
    return made


def _held(x):
    """Codes (int8) and scales (fp16) of rows [n][heads][d], as a cache holds them."""
    s = x.unflatten(-1, (-1, BLOCK)).abs().amax(-1).double() / QMAX
    s = s.float().half().clamp(max=SCALE_MAX)
    t = x.float().unflatten(-1, (-1, BLOCK)) / torch.where(s > 0, s, 1.0).float()[..., None]
    return t.round().clamp(-QMAX, QMAX).flatten(-2).to(torch.int8), s


def prepare(case, seed):
    made = _make(case, seed)
    lens, rows = made["lens"], made["rows"]
    nkv, d, page, b = case["nkv"], case["d"], case["page"], case["b"]
    need = [-(-n // page) for n in lens]
    # a pool in use: a sequence's pages lie anywhere in it
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=made["gen"], device="cuda")
    table = torch.zeros(b, max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    cache = torch.zeros(n_pages, nkv, page * d * 9 // 8, dtype=torch.uint8, device="cuda")
    st = dict(case=case, cache=cache, table=table, lens_host=lens, rows_host=rows,
              lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), row_off=None)
    # the rows' sequences and positions, for the plain form
    st["seq"] = torch.tensor([i for i, r in enumerate(rows) for _ in range(r)], device="cuda")
    st["pos"] = torch.tensor([p for n, r in zip(lens, rows) for p in range(n - r, n)], device="cuda")
    m = sum(rows)
    if len(set(rows)) > 1:
        off = [0]
        for r in rows:
            off.append(off[-1] + r)
        st["row_off"] = torch.tensor(off, dtype=torch.int32, device="cuda")
    dt = _dtype(case)
    if case["op"] == "store":
        # k | v of one stacked projection's output
        st["k"], st["v"] = made["kv"][:, 0].flatten(1), made["kv"][:, 1].flatten(1)
    else:
        for i, ((kq, ks), (vq, vs)) in enumerate(made["held"]):
            made["held"][i] = None
            _put(cache, case, table, i, torch.arange(lens[i], device="cuda"), kq, ks, vq, vs)
    if case["op"] == "attn":
        st["q"] = made["q"].flatten(1)
        st["out"] = torch.empty_like(st["q"])
    else:
        st["k_out"] = torch.empty(m, nkv * d, dtype=dt, device="cuda")
        st["v_out"] = torch.empty_like(st["k_out"])
    if own:
        from madi_amd import kv4, q8
        q8.init()
        st["kv4"] = kv4.KV4(cache, page=page, heads=nkv, dim=d)
        st["batch"] = kv4.Batch(table, st["lens"], rows=max(rows), row_off=st["row_off"], m=m,
                                len_max=max(lens))
        if case["op"] == "attn":
            st["batch"].reserve(st["kv4"], case["nh"])
    return st


# ---------------------------------------------------------------- the cache's bytes
def _views(cache, case):
    """The regions of every page and head.
    K  [page][heads][token][4][blocks][4 bytes]: word (g, b) holds elements 32 b + 8 g + 0..7,
       element 2 j in nibble j and element 2 j + 1 in nibble 4 + j.
    V  [page][heads][token / 4][16][blocks][4 bytes]: word (c, b) holds elements 32 b + c (low
       nibbles) and 32 b + 16 + c (high) of four tokens, bytes in token order 0, 2, 1, 3.
    S  [page][heads][token / 4][K, V][blocks][4 tokens] fp16."""
    t, d = case["page"], case["d"]
    nb = d // BLOCK
    k = cache[:, :, :t * d // 2].unflatten(2, (t, 4, nb, 4))
    v = cache[:, :, t * d // 2:t * d].unflatten(2, (t // 4, 16, nb, 4))
    s = cache[:, :, t * d:].view(torch.float16).unflatten(2, (t // 4, 2, nb, 4))
    return k, v, s


def _k_words(q):
    """Codes [n][heads][d] -> K bytes [n][heads][4][blocks][4]."""
    n = (q + 8).to(torch.uint8).unflatten(-1, (-1, 4, 8))  # [.., b, g, e]
    lo, hi = n[..., [0, 4, 1, 5]], n[..., [2, 6, 3, 7]]
    return (lo | (hi << 4)).transpose(-3, -2)


def _v_bytes(q):
    """Codes [n][heads][d] -> V bytes [n][heads][16][blocks]."""
    n = (q + 8).to(torch.uint8).unflatten(-1, (-1, 2, 16))  # [.., b, half, c]
    return (n[..., 0, :] | (n[..., 1, :] << 4)).transpose(-2, -1)


def _place(case, table, seq, pos):
    """Page, token within it and byte of a V word of positions `pos` of `seq`."""
    t = case["page"]
    off = pos % t
    return table[seq, pos // t].long(), off, (off & 1) * 2 + (off >> 1 & 1)


def _put(cache, case, table, seq, pos, kq, ks, vq, vs):
    """Write rows into positions `pos` of sequences `seq`."""
    k, v, s = _views(cache, case)
    page, off, tok = _place(case, table, seq, pos)
    k[page, :, off] = _k_words(kq)
    v[page, :, off // 4, :, :, tok] = _v_bytes(vq)
    s[page, :, off // 4, 0, :, off % 4] = ks
    s[page, :, off // 4, 1, :, off % 4] = vs


def _get(cache, case, table, seq, pos):
    """The rows at positions `pos` of sequences `seq` as f32 K and V [n][heads][d]."""
    k, v, s = _views(cache, case)
    page, off, tok = _place(case, table, seq, pos)
    w = k[page, :, off].transpose(-3, -2)  # [n][heads][b][g][4 bytes]
    lo, hi = w & 15, w >> 4
    kn = torch.stack([lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2],
                      lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]], -1).flatten(-2)
    w = v[page, :, off // 4, :, :, tok].transpose(-2, -1)  # [n][heads][b][16]
    vn = torch.cat([w & 15, w >> 4], -1)
    ks = s[page, :, off // 4, 0, :, off % 4]
    vs = s[page, :, off // 4, 1, :, off % 4]
    return (((kn.float() - 8) * ks.float()[..., None]).flatten(-2),
            ((vn.float() - 8) * vs.float()[..., None]).flatten(-2))


# ---------------------------------------------------------------- one pass
def _plain_quant(x):
    """The definition in torch; the borders between codes in 64 bits."""
    x = x.unflatten(-1, (-1, BLOCK))
    s = (x.abs().amax(-1).double() / QMAX).float().half().clamp(max=SCALE_MAX)
    t = x.abs().double() / torch.where(s > 0, s, 1.0).double()[..., None]
    q = (t + 0.5).floor().clamp(max=QMAX) * (s > 0)[..., None]
    return torch.where(x < 0, -q, q).flatten(-2).to(torch.int8), s


def _plain_attn(st):
    case = st["case"]
    nh, nkv, d = case["nh"], case["nkv"], case["d"]
    g, at = nh // nkv, 0
    out = st["out"]
    for i, (n, r) in enumerate(zip(st["lens_host"], st["rows_host"])):
        first = 0
        if case["causal"] and case["window"]:
            first = max(0, n - r - case["window"] + 1)
        key = torch.arange(first, n, device=out.device)
        k, v = _get(st["cache"], case, st["table"], i, key)
        q = st["q"][at:at + r].float().unflatten(1, (nkv, g, d)).permute(1, 0, 2, 3)  # [kv][r][g][d]
        pos = torch.arange(n - r, n, device=q.device)[:, None, None]
        hidden = torch.zeros(r, 1, n - first, dtype=torch.bool, device=q.device)
        if case["causal"]:
            hidden = key > pos
            if case["window"]:
                hidden = hidden | (key <= pos - case["window"])
        for h in range(nkv) if r * g * (n - first) > (1 << 16) else [slice(None)]:
            kh, vh = k[:, h], v[:, h]
            if isinstance(h, slice):
                kh, vh = kh.permute(1, 2, 0).contiguous(), vh.permute(1, 0, 2).contiguous()
                x = (q[h].flatten(1, 2) @ kh).unflatten(1, (r, g))
            else:
                x = (q[h].flatten(0, 1) @ kh.T.contiguous()).unflatten(0, (r, g))
            x = (x * (1.0 / math.sqrt(d))).masked_fill(hidden, float("-inf"))
            p = (x - x.amax(-1, keepdim=True)).exp()
            o = (p.flatten(-3, -2) @ vh).unflatten(-2, (r, g)) / p.sum(-1, keepdim=True)
            o = o.permute(1, 0, 2, 3) if isinstance(h, slice) else o[:, None]
            out[at:at + r].unflatten(1, (nkv, g, d))[:, h if isinstance(h, slice) else slice(h, h + 1)] = o.to(out.dtype)
        at += r
    return out


def run(st):
    case = st["case"]
    if own:
        from madi_amd import kv4
        if case["op"] == "attn":
            kv4.kvAttn(st["out"], st["q"], st["kv4"], st["batch"], case["nh"], causal=case["causal"],
                       window=case["window"])
            return st["out"]
        if case["op"] == "store":
            kv4.kvStore(st["kv4"], st["batch"], st["k"], st["v"])
        kv4.kvLoad(st["kv4"], st["batch"], st["k_out"], st["v_out"])
        return st["k_out"], st["v_out"]
    if case["op"] == "attn":
        return _plain_attn(st)
    at = st["table"], st["seq"], st["pos"]
    if case["op"] == "store":
        heads = (case["nkv"], case["d"])
        _put(st["cache"], case, *at, *_plain_quant(st["k"].unflatten(1, heads)),
             *_plain_quant(st["v"].unflatten(1, heads)))
    k, v = _get(st["cache"], case, *at)
    st["k_out"].copy_(k.flatten(1))
    st["v_out"].copy_(v.flatten(1))
    return st["k_out"], st["v_out"]


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    made = _make(case, seed)
    nkv, d = case["nkv"], case["d"]
    value = lambda q, s: q.double() * s.double().repeat_interleave(BLOCK, -1)
    if case["op"] == "store":
        out = []
        for x in (made["kv"][:, 0].double(), made["kv"][:, 1].double()):
            top = x.abs().reshape(-1, BLOCK).max(1).values / 7
            s = top.float().half().double().clamp(max=9352)[:, None]
            mag = torch.div(x.abs().reshape(-1, BLOCK) + s / 2, s.clamp(min=2.0 ** -30),
                            rounding_mode="floor").clamp(max=7)
            out.append((torch.sign(x).reshape(-1, BLOCK) * mag * s).reshape(-1, nkv * d))
        return tuple(out)
    if case["op"] == "load":
        back = [[value(*kv)[n - r:] for kv in held]
                for held, n, r in zip(made["held"], made["lens"], made["rows"])]
        return tuple(torch.cat([x[j] for x in back]).reshape(-1, nkv * d) for j in (0, 1))
    outs, at = [], 0
    for (k, v), n, r in zip(made["held"], made["lens"], made["rows"]):
        key, pos = torch.arange(n, device="cuda")[None], torch.arange(n - r, n, device="cuda")[:, None]
        seen = torch.ones(r, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = key <= pos
            if case["window"]:
                seen &= key > pos - case["window"]
        o = torch.empty(r, case["nh"], d, dtype=torch.float64, device="cuda")
        for h in range(nkv):
            kh, vh = value(k[0][:, h], k[1][:, h]), value(v[0][:, h], v[1][:, h])
            for j in range(h * (case["nh"] // nkv), (h + 1) * (case["nh"] // nkv)):
                x = made["q"][at:at + r, j].double() @ kh.T.contiguous() * d ** -0.5
                x = torch.where(seen, x, -math.inf)
                p = torch.softmax(x, -1)
                o[:, j] = p @ vh
        outs.append(o.reshape(r, -1))
        at += r
    return torch.cat(outs)
