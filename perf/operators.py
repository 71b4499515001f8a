"""Cases of the FP4 paged cache, the attention over it and the page operations.

``run`` makes one pass through an operator.  With ``own`` false it computes the
operators in elementary torch operations; with ``own`` true it calls
``intent_attention``.

FP4 rows: 32 channels of a row share a scale 2^e, e the smallest integer with
6 * 2^e >= max|x| held in [-14, 13]; an element is x * 2^-e rounded to the
nearest of {0, 0.5, 1, 1.5, 2, 3, 4, 6} (ties to the even code), with its sign.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "intent-attention-kernel_b200")
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_DEV = "cuda"


def _ia():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import intent_attention
    return intent_attention


# --------------------------------------------------------------------------- #
#  Cases
# --------------------------------------------------------------------------- #

def listed():
    return [
        # one decode step's rows of a low-bit serving batch (64 sequences, 8 kv heads)
        dict(name="append_step", op="append", batch=64, kv_heads=8, head_dim=128, page=16, rows=1, start=8000,
             ragged=False, dtype="bf16"),
        # ragged prompts written in one call, padded to the longest
        dict(name="append_prompt", op="append", batch=4, kv_heads=8, head_dim=128, page=64, rows=8187, start=0,
             ragged=True, dtype="f16"),
        # a short prefix taken out of the cache for a check or a move
        dict(name="read_prefix", op="read", batch=2, kv_heads=2, head_dim=64, page=32, rows=101, start=5,
             ragged=True, dtype="f32"),
        # whole contexts moved to a 16-bit cache
        dict(name="read_context", op="read", batch=8, kv_heads=8, head_dim=128, page=16, rows=32768, start=0,
             ragged=False, dtype="bf16"),
        # the CPU-runnable multi-head shape: one short sequence, latency counts
        dict(name="decode_short", op="decode", batch=1, heads=8, kv_heads=8, head_dim=64, page=16, queries=1,
             tokens=1440, ragged=False, dtype="f32"),
        # a grouped-query serving batch at 32k context
        dict(name="decode_batch", op="decode", batch=32, heads=32, kv_heads=8, head_dim=128, page=16, queries=1,
             tokens=32768, ragged=True, dtype="bf16"),
        # one long context: the cache's axis is all there is to split
        dict(name="decode_long", op="decode", batch=1, heads=32, kv_heads=8, head_dim=128, page=64, queries=1,
             tokens=524287, ragged=False, dtype="f16"),
        # draft tokens checked together, wide heads
        dict(name="decode_draft", op="decode", batch=16, heads=16, kv_heads=2, head_dim=256, page=32, queries=4,
             tokens=8001, ragged=True, dtype="bf16"),
        # differential attention: a small batch of a step
        dict(name="differential_step", op="differential", batch=4, heads=8, kv_heads=4, head_dim=128, page=16,
             queries=1, tokens=2003, ragged=True, dtype="f16"),
        # differential attention: a serving batch at 32k context
        dict(name="differential_batch", op="differential", batch=16, heads=32, kv_heads=8, head_dim=128, page=16,
             queries=1, tokens=32768, ragged=True, dtype="bf16"),
        # parallel samples of 8 prompts: share the pages, one token more each, the prompts' slots given back
        dict(name="pages_fork", op="fork", sources=8, copies=7, kv_heads=8, head_dim=128, page=16, tokens=1000),
        # a fragmented 16-bit cache packed to the lowest pages
        dict(name="pages_compact", op="compact", slots=64, kv_heads=8, pages_each=320, pages=262144, moves=98304,
             head_dim=128, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "differential", "fork", "compact"])
    if op in ("append", "read"):
        d, b, h = rng.choice([64, 128, 256]), _log(rng, 1, 64), rng.choice([1, 2, 3, 4, 8])
        rows = _log(rng, 1, max(1, min(16384, 2 ** 28 // (b * h * d * (1 if op == "read" else 4)))))
        return dict(op=op, batch=b, kv_heads=h, head_dim=d, page=rng.choice([16, 32, 64, 128]), rows=rows,
                    start=rng.choice([0, 1, 7, _log(rng, 1, 4000)]), ragged=rng.random() < 0.6,
                    dtype=rng.choice(["f32", "f16", "bf16"]))
    if op in ("decode", "differential"):
        d, b, h = rng.choice([64, 128, 256]), _log(rng, 1, 48), rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 4, 5, 7, 8, 16])
        queries = rng.choice([1, 1, 1, 2, 3, 4, 8])
        most = 2 ** 28 // (b * h * d * max(1, group * queries // 8))
        return dict(op=op, batch=b, heads=h * group, kv_heads=h, head_dim=d, page=rng.choice([16, 32, 48, 64, 128]),
                    queries=queries, tokens=_log(rng, 1, max(2, min(400000, most))), ragged=rng.random() < 0.6,
                    dtype=rng.choice(["f32", "f16", "bf16", "bf16"]))
    if op == "fork":
        return dict(op=op, sources=rng.randint(1, 16), copies=rng.randint(1, 7), kv_heads=rng.choice([1, 2, 4, 8]),
                    head_dim=rng.choice([64, 128]), page=rng.choice([8, 16, 32, 64]), tokens=_log(rng, 1, 4000))
    slots, h, each = rng.randint(1, 64), rng.choice([1, 2, 4, 8]), _log(rng, 1, 300)
    live = slots * h * each
    pages = live + _log(rng, 1, 100000)
    return dict(op=op, slots=slots, kv_heads=h, pages_each=each, pages=pages,
                moves=rng.randint(0, min(live, pages - live)), head_dim=rng.choice([64, 128]), page=16)


def _lengths(case):
    n, b = case["tokens"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [max(1, n - (5 * n * i) // (8 * b) - (7 * i) % 16) for i in range(b)]


def _starts(case):
    return [case["start"] + (3 * i) % 17 for i in range(case["batch"])]


def _counts(case):
    n, b = case["rows"], case["batch"]
    return [n - (n * i) // (2 * b) if case["ragged"] else n for i in range(b)]


def _fork_lengths(case):
    return [max(1, case["tokens"] - (5 * i) % (2 * case["page"])) for i in range(case["sources"])]


def work(case):
    op = case["op"]
    if op in ("append", "read"):
        size, d = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]], case["head_dim"]
        held, dense = d * 17 // 32, d * size
        rows = 2 * case["kv_heads"] * sum(_counts(case))
        if op == "read":
            return {"bytes": rows * (held + dense), "flops": 0}
        # written rows, and the read back of them and of the row before
        back = rows + 2 * case["kv_heads"] * sum(1 for s in _starts(case) if s)
        return {"bytes": rows * (dense + held) + back * (held + dense), "flops": 0}
    if op in ("decode", "differential"):
        size, d, m = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]], case["head_dim"], case["queries"]
        tokens = sum(_lengths(case))
        table = 4 * case["kv_heads"] * sum(-(-n // case["page"]) for n in _lengths(case))
        keys = sum(max(0, n - j) for n in _lengths(case) for j in range(m))
        per = 4 if op == "decode" else 6
        return {"bytes": 2 * case["kv_heads"] * tokens * (d * 17 // 32) + table +
                2 * case["batch"] * case["heads"] * m * d * size,
                "flops": per * d * case["heads"] * keys}
    page_bytes = 2 * 2 * case["page"] * case["head_dim"]
    if op == "fork":
        lens, each, h = _fork_lengths(case), 1 + case["copies"], case["kv_heads"]
        entries = h * sum(-(-n // case["page"]) for n in lens)
        copied = h * each * sum(1 for n in lens if n % case["page"])
        return {"bytes": copied * 2 * page_bytes + 4 * entries * (2 + 2 * case["copies"]), "flops": 0}
    entries = case["slots"] * case["kv_heads"] * case["pages_each"]
    return {"bytes": case["moves"] * 2 * page_bytes + 8 * entries + 8 * case["pages"], "flops": 0}


# --------------------------------------------------------------------------- #
#  Inputs
# --------------------------------------------------------------------------- #

def _generator(seed, what):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed * 1009 + what)
    return g


def _rows(case, seed, b, n):
    """Dense K and V rows [Ht, n, D] of one sequence: keys with a few strong channels, values near normal."""
    g = _generator(seed, 16 + 2 * b)
    h, d = case["kv_heads"], case["head_dim"]
    dt = _DTYPES[case["dtype"]]
    strong = torch.exp(0.6 * torch.randn((h, 1, d), generator=g, device=_DEV))
    k = (torch.randn((h, n, d), generator=g, device=_DEV) * strong).to(dt)
    v = torch.randn((h, n, d), generator=g, device=_DEV).to(dt)
    return k, v


def _table(case, seed, tokens):
    """Every (sequence, kv head)'s pages in no order of the pool; one page more than they need."""
    b, h = case["batch"], case["kv_heads"]
    width = -(-tokens // case["page"]) + 1
    pages = b * h * width
    perm = torch.randperm(pages, generator=_generator(seed, 3), device=_DEV)
    return perm.to(torch.int32).view(b, h, width).contiguous(), pages


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _new_cache(case, pages):
    if own:
        return _ia().Fp4Pool.allocate(pages, case["page"], case["head_dim"], device=_DEV, zero=True)
    d, ps = case["head_dim"], case["page"]
    return {x: torch.zeros((pages, ps, w), dtype=torch.uint8, device=_DEV)
            for x, w in (("kc", d // 2), ("ks", d // 32), ("vc", d // 2), ("vs", d // 32))}


def _fill(cache, case, seed, table, lengths):
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        k, v = _rows(case, seed, b, n)
        if own:
            _ia().append_fp4(cache, k[None], v[None], table[b:b + 1])
        else:
            _plain_write(cache, k, v, table[b], 0, case["page"])


def _fork_state(case, seed):
    g = _generator(seed, 5)
    h, ps, each = case["kv_heads"], case["page"], 1 + case["copies"]
    lens = _fork_lengths(case)
    width = -(-(case["tokens"] + 1) // ps) + 1
    slots = case["sources"] * each
    used = [h * (-(-n // ps)) for n in lens]
    pages = sum(used) + 2 * slots * h + 64
    perm = torch.randperm(pages, generator=g, device=_DEV).to(torch.int32)
    table = torch.full((slots, h, width), -1, dtype=torch.int32, device=_DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEV)
    at = 0
    for s, n in enumerate(lens):
        w = -(-n // ps)
        ids = perm[at:at + h * w].view(h, w)
        table[s, :, :w] = ids
        refs[ids.reshape(-1).long()] = 1
        at += h * w
    lengths = _ints(lens + [0] * (slots - len(lens)))
    src = _ints([s for s in range(case["sources"]) for _ in range(case["copies"])])
    dst = _ints(list(range(case["sources"], slots)))
    return pages, refs, table, lengths, dict(src=src, dst=dst, more=torch.ones_like(lengths),
                                             gone=_ints(list(range(case["sources"]))))


def _compact_state(case, seed):
    g = _generator(seed, 6)
    s, h, w, pages = case["slots"], case["kv_heads"], case["pages_each"], case["pages"]
    live, moves = s * h * w, case["moves"]
    low = torch.randperm(live, generator=g, device=_DEV)[:live - moves]
    high = live + torch.randperm(pages - live, generator=g, device=_DEV)[:moves]
    ids = torch.cat([low, high])
    ids = ids[torch.randperm(live, generator=g, device=_DEV)].to(torch.int32)
    table = torch.full((s, h, w + 1), -1, dtype=torch.int32, device=_DEV)
    table[:, :, :w] = ids.view(s, h, w)
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEV)
    refs[ids.long()] = 1
    lengths = _ints([w * case["page"] - (3 * i) % case["page"] for i in range(s)])
    return pages, refs, table, lengths, {}


def prepare(case, seed):
    op = case["op"]
    if op in ("append", "read"):
        starts, counts = _starts(case), _counts(case)
        last = max(starts) + case["rows"]
        table, pages = _table(case, seed, last)
        cache = _new_cache(case, pages)
        state = dict(case=case, cache=cache, table=table, starts=starts, counts=counts, positions=_ints(starts),
                     valid=_ints(counts))
        if op == "read":
            _fill(cache, case, seed, table, [s + n for s, n in zip(starts, counts)])
            return state
        back = [1 if s else 0 for s in starts]
        state["back"] = back
        state["back_positions"] = _ints([s - x for s, x in zip(starts, back)])
        state["back_valid"] = _ints([n + x for n, x in zip(counts, back)])
        rows = [_rows(case, seed, b, case["rows"]) for b in range(case["batch"])]
        state["k"] = torch.stack([r[0] for r in rows])
        state["v"] = torch.stack([r[1] for r in rows])
        # the row before each start, as an earlier step left it
        _fill_before(cache, case, seed, table, starts)
        return state
    if op in ("decode", "differential"):
        lengths = _lengths(case)
        table, pages = _table(case, seed, case["tokens"])
        cache = _new_cache(case, pages)
        _fill(cache, case, seed, table, lengths)
        state = dict(case=case, cache=cache, table=table, host_lengths=lengths, lengths=_ints(lengths))
        state.update(_queries(case, seed))
        return state
    pages, refs, table, lengths, extra = (_fork_state if op == "fork" else _compact_state)(case, seed)
    g = _generator(seed, 7)
    shape = (pages, case["page"], case["head_dim"])
    k = torch.empty(shape, dtype=torch.float16, device=_DEV).normal_(generator=g)
    v = torch.empty(shape, dtype=torch.float16, device=_DEV).normal_(generator=g)
    state = dict(case=case, k=k, v=v, refs=refs, table=table, lengths=lengths,
                 saved=(refs.clone(), table.clone(), lengths.clone()), **extra)
    if own:
        ia = _ia()
        state["pool"] = ia.PagePool(pages, case["page"], case["head_dim"], k_f16=k, v_f16=v)
        state["pages"] = ia.SequencePages(refs, table, lengths, case["page"])
    return state


def _row_before(case, seed, b):
    k, v = _rows(case, seed + 500000, b, 1)
    return k, v


def _fill_before(cache, case, seed, table, starts):
    for b, s in enumerate(starts):
        if s == 0:
            continue
        k, v = _row_before(case, seed, b)
        if own:
            _ia().append_fp4(cache, k[None], v[None], table[b:b + 1], _ints([s - 1]))
        else:
            _plain_write(cache, k, v, table[b], s - 1, case["page"])


def _queries(case, seed):
    g = _generator(seed, 4)
    shape = (case["batch"], case["heads"], case["queries"], case["head_dim"])
    q = torch.randn(shape, generator=g, device=_DEV).to(_DTYPES[case["dtype"]])
    out = {"q": q[:, :, 0].contiguous() if case["queries"] == 1 else q}
    if case["op"] == "differential":
        out["lam"] = 0.2 + 0.6 * torch.rand((case["heads"],), generator=g, device=_DEV)
        out["weight"] = 1.0 + 0.1 * torch.randn((case["head_dim"],), generator=g, device=_DEV)
    return out


# --------------------------------------------------------------------------- #
#  Plain forms (32 bits)
# --------------------------------------------------------------------------- #

def _plain_quantize(x):
    """[..., D] -> codes [..., D / 2] (even channel in the low half) and scale bytes [..., D / 32]."""
    x = x.float()
    blocks = x.view(*x.shape[:-1], -1, 32)
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1))
    e = torch.where(mantissa <= 0.75, exponent - 3, exponent - 2).clamp(-14, 13)
    y = (blocks * torch.exp2(-e.float()).unsqueeze(-1)).flatten(-2)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code | ((y < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _plain_values(codes, scales):
    lut = torch.tensor(_VALUES + tuple(-x for x in _VALUES), device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    x = lut[both.int()].view(*both.shape[:-1], -1, 32)
    return (x * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _slots(table_row, start, n, page):
    t = torch.arange(start, start + n, device=table_row.device)
    return table_row[:, t // page].long(), (t % page).expand(table_row.shape[0], n)


def _plain_write(cache, k, v, table_row, start, page):
    ids, rows = _slots(table_row, start, k.shape[1], page)
    for x, c, s in ((k, "kc", "ks"), (v, "vc", "vs")):
        codes, scales = _plain_quantize(x)
        cache[c][ids, rows] = codes
        cache[s][ids, rows] = scales


def _plain_read(cache, table_row, start, n, page):
    ids, rows = _slots(table_row, start, n, page)
    return (_plain_values(cache["kc"][ids, rows], cache["ks"][ids, rows]),
            _plain_values(cache["vc"][ids, rows], cache["vs"][ids, rows]))


def _plain_gather(state, starts, counts, most):
    case = state["case"]
    shape = (case["batch"], case["kv_heads"], most, case["head_dim"])
    k = torch.zeros(shape, dtype=_DTYPES[case["dtype"]], device=_DEV)
    v = torch.zeros_like(k)
    for b, (s, n) in enumerate(zip(starts, counts)):
        kb, vb = _plain_read(state["cache"], state["table"][b], s, n, case["page"])
        k[b, :, :n], v[b, :, :n] = kb.to(k.dtype), vb.to(v.dtype)
    return k, v


def _softmax_product(s, v):
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, (p @ v) / total, torch.zeros_like(total))


def _plain_attention(state):
    case = state["case"]
    h, d, m = case["kv_heads"], case["head_dim"], case["queries"]
    group = case["heads"] // h
    q = state["q"].view(case["batch"], h, group * m, d)
    out = torch.empty_like(q)
    for b, n in enumerate(state["host_lengths"]):
        k, v = _plain_read(state["cache"], state["table"][b], 0, n, case["page"])
        qb = q[b].float()
        last = n - m + torch.arange(m, device=_DEV).repeat(group)
        hidden = torch.arange(n, device=_DEV) > last[:, None]
        if case["op"] == "decode":
            s = (qb @ k.transpose(1, 2)) * (1.0 / math.sqrt(d))
            o = _softmax_product(s.masked_fill_(hidden, -math.inf), v)
        else:
            maps = []
            for part in (slice(0, d // 2), slice(d // 2, d)):
                s = (qb[..., part] @ k[..., part].transpose(1, 2)) * (1.0 / math.sqrt(d // 2))
                maps.append(_softmax_product(s.masked_fill_(hidden, -math.inf), v))
            lam = state["lam"].view(h, group, 1).expand(h, group, m).reshape(h, group * m, 1)
            x = maps[0] - lam * maps[1]
            o = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * state["weight"] * 0.8
        out[b] = o.to(out.dtype)
    return out.view(state["q"].shape)


def _plain_held(state, slots, page):
    """Which table entries of these slots hold pages, [n, 1, W]."""
    width = state["table"].shape[2]
    held = (state["lengths"][slots] + page - 1) // page
    return torch.arange(width, device=_DEV) < held[:, None, None]


def _plain_fork(state, src, dst, page):
    src, dst = src.long(), dst.long()
    held = _plain_held(state, src, page)
    rows = state["table"][src]
    state["table"][dst] = torch.where(held, rows, state["table"][dst])
    ids = rows[held.expand_as(rows)].long()
    state["refs"].index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    state["lengths"][dst] = state["lengths"][src]


def _plain_grow(state, more, page):
    refs, table, lengths = state["refs"], state["table"], state["lengths"]
    old, new = (lengths + page - 1) // page, (lengths + more + page - 1) // page
    at = torch.arange(table.shape[2], device=_DEV)
    fresh = ((at >= old[:, None, None]) & (at < new[:, None, None])).expand_as(table)
    open_page = (at == old[:, None, None] - 1) & ((more > 0) & (lengths % page > 0))[:, None, None]
    shared = open_page & (refs[table.clamp(min=0).long()] > 1)
    where = (fresh | shared).nonzero(as_tuple=True)
    before = table[where].long()
    copied = shared[where]
    ids = (refs == 0).nonzero()[:before.numel(), 0]
    for x in (state["k"], state["v"]):
        x[ids[copied]] = x[before[copied]]
    refs.index_add_(0, before[copied], torch.full_like(before[copied], -1, dtype=torch.int32))
    refs[ids] = 1
    table[where] = ids.to(torch.int32)
    lengths += more


def _plain_free(state, slots, page):
    slots = slots.long()
    held = _plain_held(state, slots, page)
    rows = state["table"][slots]
    ids = rows[held.expand_as(rows)].long()
    state["refs"].index_add_(0, ids, torch.full_like(ids, -1, dtype=torch.int32))
    state["table"][slots] = torch.where(held, torch.full_like(rows, -1), rows)
    state["lengths"][slots] = 0


def _plain_compact(state, page):
    refs, table = state["refs"], state["table"]
    live = refs > 0
    count = live.sum(dtype=torch.int32)
    at = torch.arange(refs.numel(), device=_DEV)
    moved, holes = (live & (at >= count)).nonzero()[:, 0], (~live & (at < count)).nonzero()[:, 0]
    for x in (state["k"], state["v"]):
        x[holes] = x[moved]
    to = at.to(torch.int32)
    to[moved] = holes.to(torch.int32)
    refs[holes] = refs[moved]
    refs[moved] = 0
    held = _plain_held(state, torch.arange(table.shape[0], device=_DEV), page)
    table.copy_(torch.where(held, to[table.clamp(min=0).long()], table))
    return count


# --------------------------------------------------------------------------- #
#  One pass
# --------------------------------------------------------------------------- #

def run(state):
    case = state["case"]
    op = case["op"]
    dt = _DTYPES.get(case.get("dtype"))
    if op == "append":
        if own:
            ia = _ia()
            ia.append_fp4(state["cache"], state["k"], state["v"], state["table"], state["positions"], state["valid"])
            return ia.read_fp4(state["cache"], state["table"], state["back_positions"], case["rows"] + 1,
                               state["back_valid"], dtype=dt)
        for b, (s, n) in enumerate(zip(state["starts"], state["counts"])):
            _plain_write(state["cache"], state["k"][b, :, :n], state["v"][b, :, :n], state["table"][b], s,
                         case["page"])
        return _plain_gather(state, [s - x for s, x in zip(state["starts"], state["back"])],
                             [n + x for n, x in zip(state["counts"], state["back"])], case["rows"] + 1)
    if op == "read":
        if own:
            return _ia().read_fp4(state["cache"], state["table"], state["positions"], case["rows"], state["valid"],
                                  dtype=dt)
        return _plain_gather(state, state["starts"], state["counts"], case["rows"])
    if op == "decode":
        if own:
            return _ia().paged_decode_fp4(state["q"], state["cache"], state["table"], state["lengths"])
        return _plain_attention(state)
    if op == "differential":
        if own:
            return _ia().differential_decode_fp4(state["q"], state["cache"], state["table"], state["lengths"],
                                                 state["lam"], norm_weight=state["weight"], eps=1e-5, out_scale=0.8)
        return _plain_attention(state)
    # the page operations change the state in place: each pass starts from the saved one
    for x, kept in zip((state["refs"], state["table"], state["lengths"]), state["saved"]):
        x.copy_(kept)
    if op == "fork":
        if own:
            ia = _ia()
            ia.fork_sequences(state["pages"], state["src"], state["dst"])
            ia.grow_sequences(state["pool"], state["pages"], state["more"])
            ia.free_sequences(state["pages"], state["gone"])
        else:
            _plain_fork(state, state["src"], state["dst"], case["page"])
            _plain_grow(state, state["more"], case["page"])
            _plain_free(state, state["gone"], case["page"])
        return state["refs"], state["table"], state["lengths"], state["k"], state["v"]
    count = _ia().compact_pages(state["pool"], state["pages"]) if own else _plain_compact(state, case["page"])
    return state["refs"], state["table"], state["lengths"], count, state["k"], state["v"]


# --------------------------------------------------------------------------- #
#  The definition in 64 bits
# --------------------------------------------------------------------------- #

def _exact_values(x):
    """What a cache holds for dense rows [..., D]."""
    x = x.double()
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 6.0))
    # log2 may land on either side of a whole number: put the border right
    e = torch.where(6.0 * torch.exp2(e - 1) >= top, e - 1, e)
    e = torch.where(6.0 * torch.exp2(e) < top, e + 1, e).clamp(-14, 13)
    scale = torch.exp2(e).expand(*e.shape[:-1], 32).flatten(-2)
    a = (x / scale).abs()
    r = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2)))
    return torch.sign(x) * r.clamp(max=6.0) * scale


def _exact_softmax(s):
    z = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    total = z.sum(-1, keepdim=True)
    return z / torch.where(total > 0, total, torch.ones_like(total))


def exact(case, seed):
    op = case["op"]
    if op in ("append", "read"):
        starts, counts = _starts(case), _counts(case)
        most = case["rows"] + (1 if op == "append" else 0)
        shape = (case["batch"], case["kv_heads"], most, case["head_dim"])
        out = [torch.zeros(shape, dtype=torch.float64, device=_DEV) for _ in range(2)]
        for b, (s, n) in enumerate(zip(starts, counts)):
            if op == "read":
                parts = [x[:, s:s + n] for x in _rows(case, seed, b, s + n)]
            else:
                parts = [x[:, :n] for x in _rows(case, seed, b, case["rows"])]
                if s:
                    parts = [torch.cat([x, y], 1) for x, y in zip(_row_before(case, seed, b), parts)]
            for o, x in zip(out, parts):
                o[b, :, :x.shape[1]] = _exact_values(x)
        return tuple(out)
    if op not in ("decode", "differential"):
        return None
    inputs = _queries(case, seed)
    b, h, m, d = case["batch"], case["kv_heads"], case["queries"], case["head_dim"]
    group = case["heads"] // h
    q = inputs["q"].double().view(b, h, group, m, d)
    out = torch.zeros((b, h, group, m, d), dtype=torch.float64, device=_DEV)
    for i, n in enumerate(_lengths(case)):
        k, v = (_exact_values(x) for x in _rows(case, seed, i, n))
        for j in range(m):
            seen = n - m + j + 1
            if seen <= 0:
                continue
            kj, vj = k[:, :seen], v[:, :seen]
            if op == "decode":
                out[i, :, :, j] = _exact_softmax(q[i, :, :, j] @ kj.mT / math.sqrt(d)) @ vj
                continue
            c = d // 2
            first = _exact_softmax(q[i, :, :, j, :c] @ kj[..., :c].mT / math.sqrt(c)) @ vj
            second = _exact_softmax(q[i, :, :, j, c:] @ kj[..., c:].mT / math.sqrt(c)) @ vj
            x = first - inputs["lam"].double().view(h, group, 1) * second
            out[i, :, :, j] = 0.8 * inputs["weight"].double() * x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    return out.view(inputs["q"].shape)
