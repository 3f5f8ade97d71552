"""Operators of a serving batch's decode step, as measurable cases: projections
with the low-rank adapters of many requests, beam search's selection over beams
and vocabulary, the reordering of beams' states (dense buffers, page tables and
the pages that have to be copied), page tables and row maps from the lengths.

    projection  out[m] = W x16[m] + scale[a] B_a (A_a x16[m]),  x16 = f16(x), W = f16(q s),
                a = adapter of row m (none below 0)
    selection   lp[w, v] = logit[w, v] - log sum_u exp logit[w, u] over the tokens that are not
                banned; candidates score[w] + lp[w, v], of a beam that is done the one (w, eos)
                with score[w]; the n largest of a group's, in order, equal ones by the lower beam, then
                token.  Where there are fewer: -inf, beam min(i, beams - 1), eos
    gather      state i := state parent[i], its first lens[parent[i]] rows
    fork        page table row i := row parent[i], with the pages' reference counts;
                copy: the first tokens of one page into another
    grow, trim  add[i] tokens appended to sequence i: free pages, lowest first, given out in the
                order of the sequences, and for each new row its sequence, position and slot; then
                taken back (a draft's tokens, or a prompt that was turned away)

`own` selects who computes: the plain torch form, or madi_amd.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32


# ---------------------------------------------------------------- the cases
def _lora(name, m, n, k, rank, adapters, seqs):
    return dict(name=name, op="lora", m=m, n=n, k=k, rank=rank, adapters=adapters, seqs=seqs)


def _select(name, groups, beams, vocab, n, dtype, ban, done):
    return dict(name=name, op="select", groups=groups, beams=beams, vocab=vocab, n=n, dtype=dtype, ban=ban, done=done)


def _gather(name, groups, beams, states, length, width, dtype, part, inplace):
    return dict(name=name, op="gather", groups=groups, beams=beams, states=states, length=length, width=width,
                dtype=dtype, part=part, inplace=inplace)


def _fork(name, groups, beams, page, max_pages, nkv, d):
    return dict(name=name, op="fork", groups=groups, beams=beams, page=page, max_pages=max_pages, nkv=nkv, d=d)


def _grow(name, b, page, max_pages, n_pages, used, add_lo, add_hi):
    return dict(name=name, op="grow", b=b, page=page, max_pages=max_pages, n_pages=n_pages, used=used,
                add_lo=add_lo, add_hi=add_hi)


def listed():
    return [
        # one decode step of 8 slots, each with an adapter of its own: latency
        _lora("lora_step_8", 8, 1280, 1280, 16, 8, 8),
        # the FFN's down projection for 8 slots of 5 beams, an adapter per slot
        _lora("lora_down_40", 40, 1280, 5120, 32, 7, 8),
        # prompts of odd lengths through the FFN's up projection
        _lora("lora_prompts_2000", 2000, 5120, 1280, 64, 12, 16),
        # one window's beam search, five beams: latency
        _select("select_1x5", 1, 5, 51866, 5, "f32", False, False),
        # 8 slots of 5 beams, twice as many candidates, tokens suppressed, some beams done
        _select("select_8x5", 8, 5, 51866, 10, "f32", True, True),
        # a large batch over a large vocabulary
        _select("select_64x8", 64, 8, 131072, 16, "f16", True, True),
        # five beams' token histories, in place
        _gather("gather_history_5", 1, 5, 1, 448, 1, "i32", 1.0, True),
        # the decoder's self-attention caches (4 layers, K and V) of 8 slots of 5 beams
        _gather("gather_caches_40", 8, 5, 8, 448, 1280, "f32", 0.6, False),
        # page tables of 8 slots of 5 beams, and their last pages
        _fork("fork_8x5", 8, 5, 64, 7, 20, 64),
        # long documents, 64 slots of 8 beams, small pages
        _fork("fork_64x8", 64, 8, 16, 1024, 8, 64),
        # a step of 48 sequences with drafts of up to five tokens
        _grow("grow_step_48", 48, 16, 512, 16384, 0.7, 0, 5),
        # 256 prompts admitted at once
        _grow("grow_prompts_256", 256, 16, 512, 131072, 0.4, 1, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lora", "lora", "select", "select", "gather", "fork", "grow"])
    if op == "lora":
        n, k = rng.choice([(1280, 1280), (3840, 1280), (5120, 1280), (1280, 5120), (2048, 1024), (1000, 640),
                           (4096, 4096)])
        m = _log(rng, 1, max(1, min(2000, (2000 * 5120 * 1280) // (n * k))))
        rank = rng.choice([8, 16, 16, 24, 32, 64, 128])
        seqs = min(m, _log(rng, 1, 64))
        return _lora("", m, n, k, min(rank, 64) if m > 1000 else rank, rng.randint(1, seqs), seqs)
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = rng.choice([51866, 51866, 1000, 32001, 100003, 131072])
        groups = _log(rng, 1, max(1, min(128, (1 << 26) // (beams * vocab))))
        return _select("", groups, beams, vocab, rng.choice([beams, 2 * beams, beams + 3]), rng.choice(["f16", "f32"]),
                       rng.random() < 0.6, rng.random() < 0.5)
    if op == "gather":
        beams = rng.choice([2, 3, 4, 5, 8, 16])
        groups, states = _log(rng, 1, 16), rng.choice([1, 2, 8, 24])
        length, width = rng.choice([224, 448, 1000, 1500]), rng.choice([1, 64, 1280, 77])
        width = max(1, min(width, (184 << 20) // (groups * beams * states * length)))
        return _gather("", groups, beams, states, length, width, rng.choice(["f32", "f16", "i32"]) if width % 2 == 0
                       else rng.choice(["f32", "i32"]), rng.choice([1.0, 0.5, 0.9]), rng.random() < 0.5)
    if op == "fork":
        beams = rng.choice([2, 3, 4, 5, 8, 16])
        return _fork("", _log(rng, 1, 512 // beams), beams, rng.choice([16, 32, 64, 256]), _log(rng, 4, 1024),
                     rng.choice([1, 2, 8]), rng.choice([64, 64, 128]))
    b = _log(rng, 1, 1024)
    page = rng.choice([16, 16, 32, 64])
    max_pages = _log(rng, 16, 512)
    n_pages = _log(rng, 4 * b, 131072)
    hi = rng.choice([1, 1, 5, _log(rng, 1, max(1, min(max_pages * page // 2, 524288 // b)))])
    return _grow("", b, page, max_pages, n_pages, rng.choice([0.1, 0.5, 0.9]), rng.choice([0, 1, hi]), hi)


# ---------------------------------------------------------------- sizes that follow from a case
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced, in an order that is not sorted."""
    step = next(s for s in (5, 7, 11, 13, 17) if math.gcd(s, n) == 1)
    return [lo + (hi - lo + 1) * (2 * ((i * step) % n) + 1) // (2 * n) for i in range(n)]


def _seq_rows(case):
    """Rows of each sequence: m in all, one at least."""
    free = case["m"] - case["seqs"]
    want = [1 + x for x in _spread(0, 9, case["seqs"])]
    out = [1 + free * w // sum(want) for w in want]
    out[0] += case["m"] - sum(out)
    return out


def _seq_adapter(case):
    """Adapter of each sequence; every adapter is used, and from two sequences more than adapters on
    one has none."""
    a, s = case["adapters"], case["seqs"]
    return [-1 if s >= a + 2 and i == s - 1 else (i * 7) % a if math.gcd(7, a) == 1 else i % a for i in range(s)]


def _grow_sizes(case):
    """Tokens held and added, per sequence."""
    b, reach = case["b"], case["max_pages"] * case["page"]
    add = [min(a, reach // 2) for a in _spread(case["add_lo"], case["add_hi"], b)]
    budget = int(case["n_pages"] * case["used"]) // b  # pages of a sequence, at most
    most = min(reach - max(add), budget * case["page"])
    return [max(0, min(most, x)) for x in _spread(most // 4, most, b)], add


def _fork_lens(case):
    reach = case["max_pages"] * case["page"]
    return [max(1, n) for n in _spread(reach // 3, reach, case["groups"])]


def _state_size(case):
    return 2 if case["dtype"] == "f16" else 4


def work(case):
    op = case["op"]
    if op == "lora":
        m, n, k, r = case["m"], case["n"], case["k"], case["rank"]
        with_one = sum(rows for rows, a in zip(_seq_rows(case), _seq_adapter(case)) if a >= 0)
        return dict(bytes=m * (k + n) * 4 + n * k * 34 // 32 + case["adapters"] * r * (n + k) * 2 + m * 4,
                    flops=2 * m * n * k + 2 * with_one * r * (n + k))
    if op == "select":
        rows = case["groups"] * case["beams"]
        ban = (case["vocab"] + 31) // 32 * 4 if case["ban"] else 0
        return dict(bytes=rows * case["vocab"] * _state_size(case) + ban + case["groups"] * case["n"] * 12,
                    flops=rows * case["vocab"] * 4)
    if op == "gather":
        state = int(case["length"] * case["part"]) * case["width"] * _state_size(case) * case["states"]
        slots = case["groups"] * case["beams"]
        return dict(bytes=slots * state * 3 // 2 if case["inplace"] else 2 * slots * state, flops=0)
    if op == "fork":
        b = case["groups"] * case["beams"]
        entries = sum(-(-n // case["page"]) for n in _fork_lens(case)) * case["beams"]
        return dict(bytes=entries * 12 + b // 2 * case["nkv"] * case["page"] * case["d"] * 9 // 8, flops=entries)
    held, add = _grow_sizes(case)
    p = case["page"]
    pages = sum(-(-(h + a) // p) - -(-h // p) for h, a in zip(held, add))
    return dict(bytes=case["b"] * 20 + pages * 16 + sum(add) * 16, flops=pages + sum(add))


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _make_lora(case, seed):
    gen = _generator(seed)
    m, n, k, r, na = case["m"], case["n"], case["k"], case["rank"], case["adapters"]
    w = (_randn(gen, n, k) / math.sqrt(k)).unflatten(1, (-1, BLOCK))
    s = (w.abs().amax(-1) / 127).half()
    q = (w / s.float()[..., None]).round().clamp(-127, 127).to(torch.int8).flatten(1)
    x = _randn(gen, m, k)
    x[:, ::97] *= 8  # a few large channels, as activations have them
    return dict(q=q, s=s, x=x, a=(_randn(gen, na, r, k) / math.sqrt(k)).half(), b=(_randn(gen, na, n, r) * 0.05).half(),
                scale=torch.rand(na, generator=gen, device="cuda") * 2 + 0.25,
                seq_adapter=_ints(_seq_adapter(case)),
                row_seq=torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), _ints(_seq_rows(case))))


def _make_select(case, seed):
    gen = _generator(seed)
    g, w, v = case["groups"], case["beams"], case["vocab"]
    logits = _randn(gen, g * w, v) * 2
    # a few tokens stand out, the same ones for a group's beams
    at = torch.randint(0, v, (g, 1, 12), generator=gen, device="cuda").expand(g, w, 12).reshape(g * w, 12)
    logits.scatter_add_(1, at, _randn(gen, g * w, 12).abs() * 3 + 4)
    # (the beams' scores are apart: a running sum of log probabilities)
    score = -torch.rand(g, w, generator=gen, device="cuda").cumsum(1) * 3 - 10
    made = dict(logits=logits.to(torch.float16 if case["dtype"] == "f16" else torch.float32), score=score,
                done=None, ban=None, banned=None)
    if case["done"]:
        made["done"] = torch.rand(g, w, generator=gen, device="cuda") < 0.2
    if case["ban"]:  # special tokens and a scattered list, one for all beams
        words = (v + 31) // 32
        banned = torch.rand(words * 32, generator=gen, device="cuda") < 0.03
        banned[v - v // 40:] = True
        made["ban"] = ((banned.view(words, 32).long() << torch.arange(32, device="cuda")).sum(1)).to(torch.int32)
    return made


def _idempotent(gen, groups, beams):
    """Parents with survivors left in place: a second pass changes nothing more."""
    alive = torch.rand(groups, beams, generator=gen, device="cuda") < 0.5
    alive[:, 0] = True
    order = torch.rand(groups, beams, beams, generator=gen, device="cuda").masked_fill(~alive[:, None], -1)
    return torch.where(alive, torch.arange(beams, device="cuda"), order.argmax(-1)).to(torch.int32)


def _make_gather(case, seed):
    gen = _generator(seed)
    g, w = case["groups"], case["beams"]
    shape = (case["states"], g * w, case["length"], case["width"])
    if case["dtype"] == "i32":
        src = torch.randint(0, 51866, shape, generator=gen, device="cuda", dtype=torch.int32)
    else:
        src = _randn(gen, *shape).to(torch.float16 if case["dtype"] == "f16" else torch.float32)
    parent = _idempotent(gen, g, w) if case["inplace"] else \
        torch.randint(0, w, (g, w), generator=gen, device="cuda", dtype=torch.int32)
    return dict(src=src, parent=parent,
                lens=torch.full((g * w,), int(case["length"] * case["part"]), dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    st = dict(case=case)
    gen = _generator(seed)
    op = case["op"]
    if op == "lora":
        st.update(_make_lora(case, seed))
        st["adapter"] = st["seq_adapter"][st["row_seq"]].contiguous()
        st["out"] = torch.empty(case["m"], case["n"], device="cuda")
        if own:
            from madi_amd import lora, q8
            q8.init()
            st["w"] = q8.upload_q8_device_repack(st["q"].cpu().numpy(), st["s"].cpu().numpy())
            st["lora"] = lora.Adapters(st["a"], st["b"], st["scale"])
            st["lora"].reserve(case["m"])
    elif op == "select":
        st.update(_make_select(case, seed))
        if own:
            from madi_amd import beam, q8
            q8.init()
            st["search"] = beam.Search(case["groups"], case["beams"], case["vocab"], n=case["n"], eos=1)
    elif op == "gather":
        st.update(_make_gather(case, seed))
        st["dst"] = st["src"] if case["inplace"] else torch.zeros_like(st["src"])
        st["dsts"], st["srcs"] = list(st["dst"]), list(st["src"])
        if own:
            from madi_amd import q8
            q8.init()
    elif op == "fork":
        _prepare_fork(st, gen)
    else:
        _prepare_grow(st, gen)
    return st


def _count(table, lens, page, n_pages):
    """Reference counts: how many table entries name each page."""
    held = torch.arange(table.shape[1], device="cuda") * page < lens[:, None]
    at = torch.where(held, table, n_pages).flatten().long()
    return torch.zeros(n_pages + 1, dtype=torch.int32, device="cuda").index_add_(
        0, at, torch.ones_like(at, dtype=torch.int32))[:n_pages].contiguous()


def _prepare_fork(st, gen):
    """Beams that share their first pages and have up to three last ones of their own."""
    case = st["case"]
    g, w, page, mp = case["groups"], case["beams"], case["page"], case["max_pages"]
    b, lens = g * w, _fork_lens(case)
    n_pages = g * mp + 4 * b
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    st["lens"] = _ints([n for n in lens for _ in range(w)])
    c = torch.arange(mp, device="cuda")
    held = -(-st["lens"] // page)[:, None]
    tail = c >= held - torch.randint(1, 4, (b, 1), generator=gen, device="cuda")
    shared = (torch.arange(b, device="cuda") // w)[:, None] * mp + c
    mine = g * mp + 4 * torch.arange(b, device="cuda")[:, None] + (held - 1 - c).clamp(0, 3)
    st["table"] = torch.where(c < held, order[torch.where(tail, mine, shared)], -1)
    st["refs"] = _count(st["table"], st["lens"], page, n_pages)
    st["parent"] = _idempotent(gen, g, w)
    # about half of the beams go on in a copy of their last page
    some = torch.rand(b, generator=gen, device="cuda") < 0.5
    last = st["table"].gather(1, (held - 1).long())[:, 0]
    fresh = order[g * mp + 4 * torch.arange(b, device="cuda") + 3]
    used = (st["lens"] - 1) % page + 1
    st["copies"] = torch.where(some[:, None], torch.stack([last, fresh, used], 1), -1).to(torch.int32)
    # (one page more than the pool: what the plain form reads and writes for a beam without a copy)
    st["cache"] = torch.randint(0, 256, (n_pages + 1, case["nkv"], page * case["d"] * 9 // 8), generator=gen,
                                device="cuda", dtype=torch.uint8)
    if own:
        from madi_amd import kv4, q8
        q8.init()
        st["kv4"] = kv4.KV4(st["cache"], page=page, heads=case["nkv"], dim=case["d"], n_pages=n_pages)
        st["pages"] = kv4.Pages(st["refs"], st["table"], st["lens"], page)


def _prepare_grow(st, gen):
    case = st["case"]
    held, add = _grow_sizes(case)
    page, n_pages, mp = case["page"], case["n_pages"], case["max_pages"]
    # (from one seed to the next other sequences have these lengths)
    perm = torch.randperm(case["b"], generator=gen, device="cuda")
    st["lens"], st["add"] = _ints(held)[perm], _ints(add)[perm]
    st["to"] = st["lens"].clone()
    n = -(-st["lens"] // page)
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    c = torch.arange(mp, device="cuda")
    at = (n.cumsum(0) - n)[:, None] + c
    st["table"] = torch.where(c < n[:, None], order[at.clamp(max=n_pages - 1)], -1)
    # a few pages more are held elsewhere (prompts kept for the next request)
    kept = torch.rand(n_pages, generator=gen, device="cuda") < 0.05
    st["refs"] = _count(st["table"], st["lens"], page, n_pages) + kept
    st["m"] = max(1, sum(add))
    if own:
        from madi_amd import kv4, q8
        q8.init()
        st["pages"] = kv4.Pages(st["refs"], st["table"], st["lens"], page, m=st["m"])


# ---------------------------------------------------------------- one pass
def _plain_lora(st):
    case = st["case"]
    na, r, n = case["adapters"], case["rank"], case["n"]
    w = (st["q"].unflatten(1, (-1, BLOCK)).float() * st["s"].float()[..., None]).half().float().flatten(1)
    x = st["x"].half().float()
    h = (x @ st["a"].float().flatten(0, 1).T.contiguous()).unflatten(1, (na, r))
    mine = st["adapter"][:, None] == torch.arange(na, device="cuda")
    h = h * (mine * st["scale"])[..., None]
    return x @ w.T.contiguous() + h.flatten(1) @ st["b"].float().permute(0, 2, 1).reshape(na * r, n)


def _plain_select(st):
    case = st["case"]
    g, w, v, n = case["groups"], case["beams"], case["vocab"], case["n"]
    x = st["logits"].float()
    token = torch.arange(v, device="cuda")
    if st["ban"] is not None:
        banned = (st["ban"][token // 32] >> (token % 32)) & 1
        x = x.masked_fill(banned.bool(), float("-inf"))
    top = x.amax(1, keepdim=True)
    lse = top.double() + (x.double() - top.double()).exp().sum(1, keepdim=True).log()
    # the n largest of each row, equal ones by the lower token: one whole number holds both
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * (1 << 32) + ((1 << 32) - 1 - token)
    at = key.topk(min(n, v), dim=1).indices
    cand = (st["score"].double().view(-1, 1) + (x.gather(1, at).double() - lse)).view(g, w, -1)
    at = at.view(g, w, -1)
    if st["done"] is not None:
        first = torch.arange(at.shape[2], device="cuda") == 0
        only = torch.where(first, st["score"].double()[..., None], float("-inf"))
        cand = torch.where(st["done"][..., None], only, cand)
        at = torch.where(st["done"][..., None], 1, at)
    best, order = cand.flatten(1).sort(dim=1, descending=True, stable=True)
    best, order = best[:, :n], order[:, :n]
    there = best > float("-inf")
    parent = torch.where(there, order // at.shape[2], torch.arange(n, device="cuda").clamp(max=w - 1))
    token = torch.where(there, at.flatten(1).gather(1, order), 1)
    return best.float(), parent.to(torch.int32), token.to(torch.int32)


def _plain_gather(st):
    case = st["case"]
    g, w = case["groups"], case["beams"]
    src = (torch.arange(g, device="cuda")[:, None] * w + st["parent"]).flatten()
    rows = torch.arange(case["length"], device="cuda") < st["lens"][src][:, None]
    st["dst"].copy_(torch.where(rows[..., None], st["src"][:, src], st["dst"]))
    return st["dst"]


def _plain_fork(st):
    case = st["case"]
    w, page, d = case["beams"], case["page"], case["d"]
    b, n_pages = st["lens"].shape[0], st["refs"].shape[0]
    src = torch.arange(b, device="cuda") // w * w + st["parent"].flatten()
    before = _count(st["table"], st["lens"], page, n_pages)
    st["lens"].copy_(st["lens"][src])
    held = torch.arange(case["max_pages"], device="cuda") * page < st["lens"][:, None]
    st["table"].copy_(torch.where(held, st["table"][src], -1))
    st["refs"] += _count(st["table"], st["lens"], page, n_pages) - before
    # tokens in whole fours; without a copy, the page past the pool onto itself
    x = torch.arange(page * d * 9 // 8, device="cuda")
    four = (st["copies"][:, 2:] + 3) // 4
    keep = torch.where(x < page * d // 2, x < four * (2 * d),
                       torch.where(x < page * d, x - page * d // 2 < four * (2 * d), x - page * d < four * (d // 2)))
    some = st["copies"][:, 0] >= 0
    a = torch.where(some, st["copies"][:, 0], n_pages).long()
    z = torch.where(some, st["copies"][:, 1], n_pages).long()
    st["cache"][z] = torch.where((keep & some[:, None])[:, None], st["cache"][a], st["cache"][z])
    return st["table"], st["lens"], st["refs"], st["cache"]


def _plain_grow(st):
    case = st["case"]
    page, mp, b, m = case["page"], case["max_pages"], case["b"], st["m"]
    lens, n_pages = st["lens"], st["refs"].shape[0]
    fits = lens + st["add"] <= mp * page
    add = torch.where(fits, st["add"], 0).long()
    old, new = -(-lens // page), -(-(lens + add) // page)
    need = new - old
    enough = (need == 0) | (need.cumsum(0) <= (st["refs"] == 0).sum())
    grown = fits & enough & (add.cumsum(0) <= m)
    add, need = add * grown, need * grown
    c = torch.arange(mp, device="cuda")
    free = torch.argsort((st["refs"] != 0).to(torch.int32), stable=True).to(torch.int32)  # the free ones first
    fresh = (c >= old[:, None]) & (c < (old + need)[:, None])
    at = (need.cumsum(0) - need - old)[:, None] + c
    st["table"].copy_(torch.where(fresh, free[at.clamp(0, n_pages - 1)], st["table"]))
    st["refs"] += _count(torch.where(fresh, st["table"], n_pages), lens + add, page, n_pages + 1)[:n_pages]
    st["lens"] += add
    end = add.cumsum(0)
    row = torch.arange(m, device="cuda")
    seq = torch.searchsorted(end, row, right=True).clamp(max=b - 1)
    pos = st["lens"][seq] - (end[seq] - row)
    there = row < end[-1]
    slot = st["table"][seq, (pos // page).clamp(0, mp - 1)].long() * page + pos % page
    off = torch.cat([end.new_zeros(1), end]).to(torch.int32)
    maps = off, torch.where(there, seq, -1).to(torch.int32), torch.where(there, pos, 0).to(torch.int32), \
        torch.where(there, slot, -1)
    # and back
    lens = torch.minimum(st["lens"], st["to"])
    gone = (c * page >= lens[:, None]) & (c * page < st["lens"][:, None])
    st["refs"] -= _count(torch.where(gone, st["table"], n_pages), st["lens"], page, n_pages + 1)[:n_pages]
    st["table"].masked_fill_(gone, -1)
    st["lens"].copy_(lens)
    return (*maps, st["table"], st["lens"], st["refs"])


def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return dict(lora=_plain_lora, select=_plain_select, gather=_plain_gather, fork=_plain_fork,
                    grow=_plain_grow)[op](st)
    if op == "lora":
        from madi_amd import lora
        lora.pprojLora(st["x"], st["w"], st["out"], case["m"], case["n"], case["k"], st["lora"], st["adapter"])
        return st["out"]
    if op == "select":
        from madi_amd import beam
        s = st["search"]
        beam.beamSelect(s, st["logits"], st["score"], done=st["done"], ban=st["ban"])
        return s.score, s.parent, s.token
    if op == "gather":
        from madi_amd import beam
        beam.beamGather(st["dsts"], st["srcs"], st["parent"], case["beams"], lens=st["lens"])
        return st["dst"]
    from madi_amd import kv4
    p = st["pages"]
    if op == "fork":
        kv4.kvFork(p, st["parent"], case["beams"])
        kv4.kvCopy(st["kv4"], st["copies"])
        return st["table"], st["lens"], st["refs"], st["cache"]
    kv4.kvGrow(p, st["add"])
    kv4.kvTrim(p, st["to"])
    return p.row_off, p.row_seq, p.row_pos, p.slot, st["table"], st["lens"], st["refs"]


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    if case["op"] == "lora":
        c = _make_lora(case, seed)
        w = (c["q"].double() * c["s"].double().repeat_interleave(BLOCK, 1)).half().double()
        x = c["x"].half().double()
        out = x @ w.T.contiguous()
        for i in range(case["seqs"]):
            a, rows = int(c["seq_adapter"][i]), c["row_seq"] == i
            if a >= 0:
                h = x[rows] @ c["a"][a].double().T.contiguous()
                out[rows] += c["scale"][a].double() * (h @ c["b"][a].double().T.contiguous())
        return out
    if case["op"] == "select":
        c = _make_select(case, seed)
        g, w, v, n = case["groups"], case["beams"], case["vocab"], case["n"]
        scores, parents, tokens = [], [], []
        for i in range(g):
            x = c["logits"][i * w:(i + 1) * w].double()
            if c["ban"] is not None:
                bits = (c["ban"].long()[:, None] >> torch.arange(32, device="cuda")) % 2 == 1
                x[:, bits.reshape(-1)[:v]] = -math.inf
            x = c["score"][i].double()[:, None] + torch.log_softmax(x, 1)
            if c["done"] is not None:
                x[c["done"][i]] = -math.inf
                x[:, 1] = torch.where(c["done"][i], c["score"][i].double(), x[:, 1])
            best, order = torch.sort(x.reshape(-1), descending=True, stable=True)
            best = torch.cat([best, best.new_full((n,), -math.inf)])[:n]
            order = torch.cat([order, order.new_zeros(n)])[:n]
            none = torch.isinf(best)
            scores.append(best)
            parents.append(torch.where(none, torch.arange(n, device="cuda").clamp(max=w - 1), order // v))
            tokens.append(torch.where(none, 1, order % v))
        return torch.stack(scores), torch.stack(parents).to(torch.int32), torch.stack(tokens).to(torch.int32)
    if case["op"] == "gather" and case["dtype"] != "i32":
        c = _make_gather(case, seed)
        out = c["src"].double() if case["inplace"] else torch.zeros_like(c["src"], dtype=torch.float64)
        for i in range(case["groups"] * case["beams"]):
            j = i - i % case["beams"] + int(c["parent"].view(-1)[i])
            n = int(c["lens"][j])
            out[:, i, :n] = c["src"][:, j, :n].double()
        return out
    return None  # (whole numbers)
