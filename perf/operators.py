"""Cases and plain forms of the page-sharing operators, and the calls a user makes of them.

``decode``   decode attention for groups of sequences that share a prefix
``copy``     copying pages of a cache
``fork``     restarting the children of a set of prompts: release, fork, reserve (copy on write)
``compact``  moving the live pages of a pool to its lowest ids

The plain forms are elementary torch operations in 32 bits, rounded once at the end.
"""

import random

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_MAXCODE = {"int8": 127.0, "e4m3": 448.0}


# --------------------------------------------------------------------------- cases
def _decode(name, dtype, q, groups, batch, prefix, suffix, ragged, heads, kv_heads, dim, page, lay):
    return {"name": name, "op": "decode", "dtype": dtype, "q": q, "groups": groups, "batch": batch, "prefix": prefix,
            "suffix": suffix, "ragged": ragged, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "lay": lay}


def _pages(name, op, dtype, pool, count, rows, kv_heads, dim, page, lay, length=0, tokens=1):
    return {"name": name, "op": op, "dtype": dtype, "pool": pool, "count": count, "rows": rows, "kv_heads": kv_heads,
            "dim": dim, "page": page, "lay": lay, "length": length, "tokens": tokens}


def listed():
    return [
        # Four samples of one short prompt, just begun: launch latency is what counts.
        _decode("decode_4_samples", "fp16", "fp16", 1, 4, 512, 16, False, 32, 8, 128, 16, 1),
        # A chat service: 64 conversations behind one system prompt with tools and examples.
        _decode("decode_system_prompt", "bf16", "bf16", 1, 64, 8192, 1024, False, 32, 8, 128, 16, 2),
        # Several prompts sampled a different number of times (one only once), small heads, odd lengths.
        _decode("decode_ragged_groups", "fp16", "fp16", 7, 61, 3001, 499, True, 8, 2, 64, 8, 3),
        # Many questions about one document held in an 8-bit cache.
        _decode("decode_document_int8", "int8", "fp16", 1, 128, 16384, 512, False, 32, 8, 128, 32, 4),
        # A few documents of unequal length, each with its own questions, e4m3 cache.
        _decode("decode_documents_e4m3", "e4m3", "bf16", 4, 33, 16384, 700, True, 32, 8, 128, 32, 5),
        # Eight continuations of one very long context.
        _decode("decode_long_context", "fp16", "fp16", 1, 8, 131072, 2048, False, 64, 8, 128, 64, 6),
        # The tail pages of a few beams.
        _pages("copy_4_pages", "copy", "fp16", 64, 4, 0, 8, 128, 16, 7),
        # Half of a pool duplicated, as when a set of sequences moves to other pages.
        _pages("copy_half_pool", "copy", "bf16", 8192, 4000, 0, 8, 128, 16, 8),
        # One prompt sampled four times.
        _pages("fork_4_samples", "fork", "fp16", 512, 1, 4, 8, 128, 16, 9, 700, 1),
        # Eight long prompts, each with 32 samples, room for 40 more tokens each.
        _pages("fork_256_samples", "fork", "bf16", 8192, 8, 256, 8, 128, 16, 10, 16000, 40),
        # A small pool after some sequences ended.
        _pages("compact_small", "compact", "bf16", 509, 200, 5, 8, 128, 16, 11),
        # A large pool, two fifths live, before its upper part is given back.
        _pages("compact_large", "compact", "fp16", 8192, 3277, 96, 8, 128, 16, 12),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    lay = rng.randrange(1 << 30)
    op = rng.choice(["decode", "decode", "decode", "copy", "fork", "compact"])
    # Page operations move bytes whatever they stand for: 16-bit caches here.
    dtype = rng.choice(["fp16", "bf16", "int8", "e4m3"] if op == "decode" else ["fp16", "bf16"])
    page = rng.choice([8, 16, 32, 48, 64])
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    if op == "decode":
        group = rng.choice([1, 2, 4, 5, 8])
        batch = _log(rng, 2, 128)
        groups = rng.choice([1, 1, max(1, batch // 9), max(1, batch // 3)])
        # At most what the largest listed case reads and computes.
        most = min(131072, 131072 * 8 * 8 // (batch * group), 131072 // groups)
        prefix = _log(rng, 64, max(65, most))
        q = dtype if dtype in ("fp16", "bf16") else rng.choice(["fp16", "bf16"])
        c = _decode("", dtype, q, groups, batch, prefix, _log(rng, 1, 1024), rng.random() < 0.7, kv * group, kv, dim,
                    page, lay)
    elif op == "copy":
        pool = _log(rng, 16, 8192 * 16 // max(16, page))
        c = _pages("", "copy", dtype, pool, rng.randint(1, max(1, pool // 2 - 1)), 0, kv, dim, page, lay)
    elif op == "fork":
        prompts, samples, length = _log(rng, 1, 8), _log(rng, 1, 32), _log(rng, 1, 16000 * page // 64)
        tokens = rng.choice([1, 1, 7, 40])
        pool = prompts * -(-length // page) + prompts * samples * (1 + -(-(tokens + page) // page)) + 5
        c = _pages("", "fork", dtype, pool, prompts, prompts * samples, kv, dim, page, lay, length, tokens)
    else:
        pool = _log(rng, 16, 8192 * 16 // max(16, page))
        rows = _log(rng, 1, 64)
        c = _pages("", "compact", dtype, pool, max(1, int(pool * rng.uniform(0.1, 0.9))), rows, kv, dim, page, lay)
    del c["name"]
    return c


# --------------------------------------------------------------------------- shapes that follow from a case
def _layout(case):
    """Group sizes, shared tokens (whole pages) and total lengths of a decode case."""
    r = random.Random(case["lay"])
    n, batch = case["groups"], case["batch"]
    if case["ragged"]:
        cuts = sorted(r.sample(range(1, batch), n - 1)) if n > 1 else []
    else:
        cuts = [batch * i // n for i in range(1, n)]
    edges = [0] + cuts + [batch]
    sizes = [b - a for a, b in zip(edges, edges[1:])]
    shared, lens = [], []
    for i, size in enumerate(sizes):
        tokens = case["prefix"] if i == 0 or not case["ragged"] else r.randint(1, case["prefix"])
        tokens = tokens // case["page"] * case["page"]
        shared.append(tokens)
        for _ in range(size):
            own_tokens = r.randint(0 if case["ragged"] else 1, case["suffix"])
            lens.append(max(1, tokens + own_tokens))
    return sizes, shared, lens


def _prompt_lengths(case):
    r = random.Random(case["lay"])
    return [case["length"] if i == 0 else r.randint(1, case["length"]) for i in range(case["count"])]


def _page_bytes(case):
    return 2 * case["page"] * case["kv_heads"] * case["dim"] * 2  # K and V, 16 bits


def work(case):
    """Each input read once and each output written once."""
    page = case["page"]
    if case["op"] == "decode":
        sizes, shared, lens = _layout(case)
        stored = sum(shared)
        entries = sum(s // page for s in shared)
        at = 0
        for size, s in zip(sizes, shared):
            for n in lens[at:at + size]:
                stored += n - s
                entries += -(-(n - s) // page)
            at += size
        eb = 2 if case["dtype"] in ("fp16", "bf16") else 1
        kv = stored * 2 * case["kv_heads"] * case["dim"] * eb
        scales = entries * 8 * case["kv_heads"] if eb == 1 else 0
        rows = 2 * case["batch"] * case["heads"] * case["dim"] * 2
        return {"bytes": kv + scales + rows + 4 * entries,
                "flops": 4 * case["heads"] * case["dim"] * sum(lens)}
    if case["op"] == "copy":
        return {"bytes": case["count"] * (2 * _page_bytes(case) + 8), "flops": 0}
    if case["op"] == "fork":
        lens = _prompt_lengths(case)
        samples = case["rows"] // case["count"]
        pages = [-(-n // page) for n in lens]
        copied = sum(samples for n in lens if n % page)
        fresh = sum(samples * (-(-(n + case["tokens"]) // page) - p) for n, p in zip(lens, pages))
        # Source rows read, child rows written, the pool's counts read, those of the pages involved written, tails copied.
        table = 4 * (sum(pages) + samples * sum(pages) + fresh)
        counts = 4 * case["pool"] + 4 * (sum(pages) + copied + fresh)
        return {"bytes": table + counts + copied * 2 * _page_bytes(case), "flops": 0}
    live = case["count"]
    moved = _movers(case)
    return {"bytes": 8 * case["pool"] + 8 * live + moved * 2 * _page_bytes(case), "flops": 0}


def _movers(case):
    """Live pages of a compact case that lie above the live count."""
    live, pool = case["count"], case["pool"]
    return min(live, pool - live) * 2 // 3


# --------------------------------------------------------------------------- inputs
def _store(case, gen, pages):
    """K, V (and scales) of a pool: N(0, 1) values, 8-bit ones scaled per (page, KV head)."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).float()
        out.append(x)
    return out


def _quantise(x, dtype):
    if dtype in ("fp16", "bf16"):
        return x.to(_DTYPES[dtype]), None
    top = _MAXCODE[dtype]
    scale = x.abs().amax(dim=(1, 3)) / torch.full((), top, device=x.device)
    y = x / scale[:, None, :, None]
    y = y.round() if dtype == "int8" else y
    return y.clamp(-top, top).to(_DTYPES[dtype]), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + case["lay"] % 7919)
    host = np.random.default_rng([seed, case["lay"]])
    s = {"case": case, "own": own}
    if case["op"] == "decode":
        _prepare_decode(case, gen, host, s)
    else:
        _prepare_pages(case, gen, host, s)
    if own:
        _prepare_own(case, s)
    return s


def _prepare_decode(case, gen, host, s):
    sizes, shared, lens = _layout(case)
    page = case["page"]
    width = max(-(-n // page) for n in lens)
    need = sum(p // page for p in shared)
    at = 0
    for size, p in zip(sizes, shared):
        need += sum(-(-n // page) - p // page for n in lens[at:at + size])
        at += size
    pool = need + 3
    ids = host.permutation(pool).astype(np.int32)
    table = np.full((case["batch"], width), -1, np.int32)
    at, row, first = 0, 0, []
    for size, p in zip(sizes, shared):
        common = ids[at:at + p // page]
        at += p // page
        for i in range(size):
            mine = -(-lens[row] // page) - p // page
            table[row, :p // page] = common
            table[row, p // page:p // page + mine] = ids[at:at + mine]
            at += mine
            if i == 0:
                first.append(int(table[row, 0]))
            row += 1
    k, v = _store(case, gen, pool)
    q = torch.randn((case["batch"], case["heads"], case["dim"]), generator=gen, device="cuda")
    # In every other KV head the first token draws much of the attention, as first tokens do in trained models.
    lean = torch.randn((case["kv_heads"], case["dim"]), generator=gen, device="cuda")
    lean[1::2] = 0.0
    q = q + 0.5 * lean.repeat_interleave(case["heads"] // case["kv_heads"], 0)
    at = torch.tensor(first, device="cuda")
    k[at, 0] += 1.5 * lean
    s["q"] = q.to(_DTYPES[case["q"]])
    s["k"], s["k_scale"] = _quantise(k, case["dtype"])
    s["v"], s["v_scale"] = _quantise(v, case["dtype"])
    s["table"] = torch.from_numpy(table).cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["sizes"], s["shared"], s["host_lens"] = sizes, shared, lens


def _prepare_pages(case, gen, host, s):
    pool, page = case["pool"], case["page"]
    k, v = _store(case, gen, pool)
    s["k"], s["k_scale"] = _quantise(k, case["dtype"])
    s["v"], s["v_scale"] = _quantise(v, case["dtype"])
    if case["op"] == "copy":
        ids = host.permutation(pool).astype(np.int32)
        s["src"] = torch.from_numpy(ids[:case["count"]].copy()).cuda()
        s["dst"] = torch.from_numpy(ids[case["count"]:2 * case["count"]].copy()).cuda()
        return
    refs = np.zeros(pool, np.int32)
    if case["op"] == "fork":
        lens = _prompt_lengths(case)
        width = -(-(max(lens) + case["tokens"]) // page)
        prompts, rows = case["count"], case["rows"]
        table = np.full((prompts + rows, width), -1, np.int32)
        ids = host.permutation(pool).astype(np.int32)
        at = 0
        for i, n in enumerate(lens):
            p = -(-n // page)
            table[i, :p] = ids[at:at + p]
            refs[ids[at:at + p]] = 1
            at += p
        owned = np.array([-(-n // page) for n in lens] + [0] * rows, np.int32)
        seq = np.array(lens + [0] * rows, np.int32)
        s["src"] = torch.from_numpy(np.repeat(np.arange(prompts, dtype=np.int32), rows // prompts)).cuda()
        s["dst"] = torch.arange(prompts, prompts + rows // prompts * prompts, dtype=torch.int32, device="cuda")
    else:
        live, up = case["count"], _movers(case)
        low = host.permutation(live)[:live - up]
        high = live + host.permutation(pool - live)[:up]
        ids = host.permutation(np.concatenate([low, high])).astype(np.int32)
        rows = min(case["rows"], live)
        cuts = [live * i // rows for i in range(rows + 1)]
        owned = np.diff(cuts).astype(np.int32)
        width = int(owned.max()) + 2
        table = np.full((rows, width), -1, np.int32)
        for r in range(rows):
            table[r, :owned[r]] = ids[cuts[r]:cuts[r + 1]]
            # Rows after the first share the page that the first begins with.
            if r and owned[r] + 1 < width:
                table[r, 1:owned[r] + 1] = table[r, :owned[r]].copy()
                table[r, 0] = table[0, 0]
                owned[r] += 1
        np.add.at(refs, table[table >= 0], 1)
        seq = (owned * page - host.integers(0, page, rows)).astype(np.int32)
    s["table"] = torch.from_numpy(table).cuda()
    s["lens"] = torch.from_numpy(seq).cuda()
    s["owned"] = torch.from_numpy(owned).cuda()
    s["refs"] = torch.from_numpy(refs).cuda()


def _prepare_own(case, s):
    from flashattntile_b200 import PagedKVCache

    if case["op"] == "copy":
        table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
        lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        table, lens = s["table"], s["lens"]
    s["cache"] = PagedKVCache(s["k"], s["v"], table, lens, case["page"])
    s["scales"] = None if s["k_scale"] is None else {"k": s["k_scale"], "v": s["v_scale"]}
    if case["op"] == "decode":
        from flashattntile_b200.kernels.shared_prefix import find_shared_prefix

        s["plan"] = find_shared_prefix(s["cache"], s["sizes"])
    elif case["op"] != "copy":
        from flashattntile_b200.page_pool import PagePool

        s["pages"] = PagePool(s["cache"], scales=s["scales"], refs=s["refs"], owned=s["owned"])


# --------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if state["own"] else _run_plain(state)


def _run_own(s):
    from flashattntile_b200 import value_checks

    case = s["case"]
    with value_checks(False):  # as a serving loop runs: no host read-back, device-side checks only
        if case["op"] == "decode":
            from flashattntile_b200.kernels.shared_prefix import shared_prefix_decode_attention

            return shared_prefix_decode_attention(s["q"], s["cache"], s["plan"], scales=s["scales"])
        if case["op"] == "copy":
            from flashattntile_b200.paging import copy_pages

            copy_pages(s["cache"], s["src"], s["dst"], scales=s["scales"])
            return _stored(s)
        pages = s["pages"]
        if case["op"] == "fork":
            pages.release(s["dst"])
            pages.fork(s["src"], s["dst"])
            pages.reserve(case["tokens"], rows=s["dst"])
            return [pages.cache.page_table, pages.cache.seq_lens, pages.owned, pages.refs] + _stored(s)
        new = pages.compact(in_place=False)
        return [new.cache.page_table, new.refs, new.live] + _stored(s)


def _stored(s):
    return [s["k"], s["v"]]


def _run_plain(s):
    op = s["case"]["op"]
    if op == "decode":
        return _plain_decode(s)
    if op == "copy":
        _plain_copy(s, s["src"].long(), s["dst"].long())
        return _stored(s)
    if op == "fork":
        return _plain_fork(s)
    return _plain_compact(s)


def _read(s, which, ids):
    """Tokens of whole pages in 32 bits: [tokens, kv_heads, dim]."""
    x = s[which][ids].float()
    if s[which + "_scale"] is not None:
        x = x * s[which + "_scale"][ids][:, None, :, None]
    return x.reshape(-1, *x.shape[2:])


def _plain_decode(s):
    case = s["case"]
    page, hkv, dim = case["page"], case["kv_heads"], case["dim"]
    group = case["heads"] // hkv
    scale = dim ** -0.5
    out = torch.empty_like(s["q"])
    at = 0
    for size, shared in zip(s["sizes"], s["shared"]):
        rows = slice(at, at + size)
        q = s["q"][rows].float().reshape(size, hkv, group, dim)
        lens = s["host_lens"][at:at + size]
        wide = max(-(-n // page) for n in lens) - shared // page
        scores, values = [], []
        if shared:
            ids = s["table"][at, :shared // page].long()
            k, v = _read(s, "k", ids), _read(s, "v", ids)
            scores.append(torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, size * group, dim), k.permute(1, 2, 0))
                          .reshape(hkv, size, group, -1).permute(1, 0, 2, 3) * scale)
            values.append(v)
        if wide:
            ids = s["table"][rows, shared // page:shared // page + wide].long().clamp_min(0)
            k = _read(s, "k", ids.reshape(-1)).reshape(size, wide * page, hkv, dim)
            v = _read(s, "v", ids.reshape(-1)).reshape(size, wide * page, hkv, dim)
            x = torch.matmul(q, k.permute(0, 2, 3, 1)) * scale
            held = torch.arange(wide * page, device=x.device)[None] < (s["lens"][rows] - shared)[:, None]
            scores.append(torch.where(held[:, None, None, :], x, torch.full_like(x, float("-inf"))))
            values.append(v)
        top = scores[0].amax(-1, keepdim=True)
        for x in scores[1:]:
            top = torch.maximum(top, x.amax(-1, keepdim=True))
        total, mixed = 0.0, 0.0
        for i, x in enumerate(scores):
            p = torch.exp(x - top)
            total = total + p.sum(-1, keepdim=True)
            v = values[i]
            if v.dim() == 3:
                y = torch.matmul(p.permute(1, 0, 2, 3).reshape(hkv, size * group, -1), v.permute(1, 0, 2))
                mixed = mixed + y.reshape(hkv, size, group, dim).permute(1, 0, 2, 3)
            else:
                mixed = mixed + torch.matmul(p, v.permute(0, 2, 1, 3))
        out[rows] = (mixed / total).reshape(size, case["heads"], dim).to(out.dtype)
        at += size
    return out


def _plain_copy(s, src, dst):
    for x in _stored(s):
        x[dst] = x[src]


def _plain_fork(s):
    page, tokens = s["case"]["page"], s["case"]["tokens"]
    table, lens, owned, refs = s["table"], s["lens"], s["owned"], s["refs"]
    src, dst = s["src"].long(), s["dst"].long()
    pool, width = refs.numel(), table.shape[1]
    cols = torch.arange(width, device=table.device)[None]

    def count(entries, held, by):
        """refs of the held entries += by (the others go to a spare count)."""
        spare = torch.cat([refs, refs.new_zeros(1)])
        spare.index_add_(0, torch.where(held, entries, pool).reshape(-1).long(),
                         torch.full((entries.numel(),), by, dtype=refs.dtype, device=refs.device))
        refs.copy_(spare[:pool])

    # release
    old = table[dst]
    count(old, cols < owned[dst][:, None], -1)
    table[dst], lens[dst], owned[dst] = -1, 0, 0
    # fork
    used = torch.div(lens[src] + page - 1, page, rounding_mode="floor")
    held = cols < used[:, None]
    new = torch.where(held, table[src], -1)
    count(new, held, 1)
    table[dst], lens[dst], owned[dst] = new, lens[src], used.to(owned.dtype)
    # reserve: a shared tail page is copied (its last sharer keeps it when all of them are here), then new pages
    tail_at = torch.div(lens[dst], page, rounding_mode="floor")
    part = lens[dst] % page != 0
    tail = table[dst, tail_at.clamp_max(width - 1).long()]
    same = (tail[:, None] == tail[None]) & part[:, None] & part[None]
    here = same.sum(1)
    order = torch.arange(dst.numel(), device=dst.device)
    last = (torch.where(same, order[None], -1).amax(1) == order)
    at_tail = torch.where(part, tail, 0).long()
    moves = part & ~((refs[at_tail] == here) & last)
    wanted = torch.div(lens[dst] + tokens + page - 1, page, rounding_mode="floor")
    fresh = (wanted - owned[dst]).clamp_min(0)
    need = moves.to(torch.int64) + fresh
    offset = need.cumsum(0) - need
    free = refs == 0
    rank = free.to(torch.int64).cumsum(0) - 1
    ids = torch.full((pool + 1,), -1, dtype=torch.int64, device=refs.device)
    ids[torch.where(free, rank, pool)] = torch.where(free, torch.arange(pool, device=refs.device), -1)
    to = torch.where(moves, ids[offset.clamp_max(pool - 1)], at_tail)
    _plain_copy(s, at_tail, to)
    count(at_tail, moves, -1)
    count(to, moves, 1)
    here_table = table[dst]
    take = moves[:, None] & (cols == tail_at[:, None])
    here_table = torch.where(take, to[:, None].to(table.dtype), here_table)
    nth = offset[:, None] + moves[:, None].to(torch.int64) + cols - owned[dst][:, None]
    grow = (cols >= owned[dst][:, None]) & (cols < wanted[:, None])
    got = ids[torch.where(grow, nth, 0).clamp(0, pool - 1)].to(table.dtype)
    here_table = torch.where(grow, got, here_table)
    count(here_table, grow, 1)
    table[dst] = here_table
    owned[dst] = torch.maximum(owned[dst], wanted.to(owned.dtype))
    return [table, lens, owned, refs] + _stored(s)


def _plain_compact(s):
    table, refs = s["table"], s["refs"]
    pool = refs.numel()
    ids = torch.arange(pool, device=refs.device)
    live = refs > 0
    count = live.sum()
    moves, hole = live & (ids >= count), ~live & (ids < count)

    def in_order(mask):
        listed_ids = torch.full((pool + 1,), pool, dtype=torch.int64, device=refs.device)
        listed_ids[torch.where(mask, mask.to(torch.int64).cumsum(0) - 1, pool)] = ids
        return listed_ids[:pool]

    held = ids < moves.sum()
    source = torch.cat([ids, ids.new_zeros(1)])
    source[torch.where(held, in_order(hole), pool)] = in_order(moves) % pool
    target = torch.cat([ids, ids.new_zeros(1)])
    target[torch.where(held, in_order(moves), pool)] = in_order(hole) % pool
    for x in _stored(s):
        x.copy_(x[source[:pool]])
    new_table = torch.where(table >= 0, target[table.clamp_min(0).long()].to(table.dtype), table)
    new_refs = torch.where(ids < count, refs[source[:pool]], 0)
    return [new_table, new_refs, count.to(torch.int32).reshape(1)] + _stored(s)


# --------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    """The decode cases by definition: one softmax per (sequence, head) over all of its tokens, in 64 bits."""
    if case["op"] != "decode":
        return None  # copies and whole numbers
    s = prepare(case, seed)
    page, hkv, dim = case["page"], case["kv_heads"], case["dim"]
    group = case["heads"] // hkv
    out = torch.empty((case["batch"], case["heads"], dim), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["host_lens"]):
        ids = s["table"][b, :-(-n // page)].long()
        for h in range(hkv):
            k, v = s["k"][ids, :, h].double(), s["v"][ids, :, h].double()
            if s["k_scale"] is not None:
                k = k * s["k_scale"][ids, h].double()[:, None, None]
                v = v * s["v_scale"][ids, h].double()[:, None, None]
            k, v = k.reshape(-1, dim)[:n], v.reshape(-1, dim)[:n]
            heads = slice(h * group, (h + 1) * group)
            x = s["q"][b, heads].double() @ k.T / dim ** 0.5
            out[b, heads] = torch.softmax(x, -1) @ v
    return out
