"""Cases of two families of operators of the serving path, in plain torch and through the framework:

* attention of a decode batch (one query per sequence) whose sequences share long prefixes: the
  sequences of a group have the same pages at the head of their block tables;
* the pages of the KV cache [2, layers, pages, page, kv heads, 128]: copies between pages ("copy"), the
  forks of sequences into the rows of others ("fork"), the turnover of finished sequences for new ones
  ("turnover": free + take) and the compaction of a cache with holes ("compact").  Tables are int32
  [rows, width] (-1 empty), lengths int32 [rows], reference counts int32 [pages] (0 is a free page).
"""
import math

import torch

own = False

HD = 128


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # four samples of one short prompt: the smallest call, where latency counts
        dict(name="attn_4_samples", op="attn", B=4, groups=1, Hq=16, Hkv=8, page=256, prefix=512, own_max=96, alone=0),
        # a system prompt of 2k tokens before 32 conversations (heads of the 8B model)
        dict(name="attn_32_chats", op="attn", B=32, groups=1, Hq=32, Hkv=8, page=256, prefix=2048, own_max=700, alone=0),
        # a batch of 256 with prefix-cache hits in 9 groups of different sizes and lengths,
        # 40 sequences that share nothing; 5 query heads to a kv head
        dict(name="attn_256_mixed", op="attn", B=256, groups=9, Hq=40, Hkv=8, page=256, prefix=4096, own_max=1300, alone=40),
        # 256 sequences behind one document of 8k tokens
        dict(name="attn_256_document", op="attn", B=256, groups=1, Hq=32, Hkv=8, page=256, prefix=8192, own_max=1024, alone=0),
        # one page to one page, a rank's share (one kv head) of the smaller model
        dict(name="copy_1_page", op="copy", layers=28, pages=64, page=256, Hkv=1, n=1, ragged=False),
        # whole and part pages of all 36 layers of the 8B model
        dict(name="copy_24_pages", op="copy", layers=36, pages=96, page=256, Hkv=8, n=24, ragged=True),
        # a second sample of one sequence, a rank's share of the heads
        dict(name="fork_1", op="fork", layers=28, pages=256, page=256, Hkv=1, rows=16, width=16, n=1, max_len=2000),
        # a beam step: 32 losers leave their rows to forks of the winners
        dict(name="fork_32_beams", op="fork", layers=36, pages=224, page=256, Hkv=4, rows=64, width=8, n=32, max_len=1200),
        # one sequence ends, one begins
        dict(name="turnover_1", op="turnover", pages=512, page=256, rows=32, width=32, n=1, max_len=3000),
        # half of a batch of 256 ends at once, over a cache of 16k pages
        dict(name="turnover_128", op="turnover", pages=16384, page=256, rows=256, width=128, n=128, max_len=14000),
        # a few holes in a small cache
        dict(name="compact_small", op="compact", layers=28, pages=64, page=256, Hkv=1, rows=16, width=8, gone=3, max_len=700),
        # the 8B model's cache after many of its sequences have left
        dict(name="compact_large", op="compact", layers=36, pages=120, page=256, Hkv=8, rows=48, width=8, gone=24, max_len=800),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "copy", "fork", "turnover", "compact"])
    page = rng.choice([256, 256, 256, 512])
    if op == "attn":
        B = _spread(rng, 2, 256)
        Hkv = rng.choice([1, 2, 4, 8])
        groups = min(max(1, B // 2), _spread(rng, 1, 24))
        return dict(op=op, B=B, groups=groups, Hq=Hkv * rng.choice([1, 2, 3, 4, 5, 8]), Hkv=Hkv, page=page,
                    prefix=_spread(rng, 300, 8000), own_max=_spread(rng, 1, 1000),
                    alone=rng.choice([0, rng.randint(0, max(0, B - 2 * groups))]))
    layers, Hkv = rng.choice([1, 7, 28, 36]), rng.choice([1, 2, 3, 8])
    if op == "copy":
        n = _spread(rng, 1, 20)
        pages = 2 * n + rng.randint(1, 40)
        layers = max(1, min(layers, int(3e9 / (pages * page * Hkv * HD * 4))))
        return dict(op=op, layers=layers, pages=pages, page=page, Hkv=Hkv, n=n,
                    ragged=rng.random() < 0.6)
    rows = _spread(rng, 4, 48)
    if op == "turnover":
        rows = _spread(rng, 4, 256)
        width = _spread(rng, 4, 64)
        return dict(op=op, pages=rows * width + rng.randint(0, 999), page=page, rows=rows, width=width,
                    n=_spread(rng, 1, rows // 2), max_len=rng.randint(page, width * page))
    max_len = rng.randint(page // 2, 3 * page)
    pages = rows * -(-max_len // page) + rng.randint(1, rows if op == "fork" else 9)
    layers = max(1, min(layers, int(3e9 / (pages * page * Hkv * HD * 4))))
    if op == "fork":
        return dict(op=op, layers=layers, pages=pages, page=page, Hkv=Hkv, rows=rows, width=4,
                    n=_spread(rng, 1, rows // 2), max_len=max_len)
    return dict(op=op, layers=layers, pages=pages, page=page, Hkv=Hkv, rows=rows, width=4,
                gone=_spread(rng, 1, rows - 2), max_len=max_len)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _attn_shape(case):
    """(members' group per sequence, shared pages per group, keys per sequence): from the case alone, so
    that work() knows them too; the lengths are ragged and the members of the groups lie mixed."""
    g = torch.Generator().manual_seed(1000003 * case["B"] + 7919 * case["prefix"] + 31 * case["own_max"] + case["groups"])
    B, n, page = case["B"], case["groups"], case["page"]
    weight = torch.rand(n, generator=g) + 0.2
    group = torch.multinomial(weight, B, replacement=True, generator=g)
    group[:min(B, 2 * n)] = torch.arange(min(B, 2 * n)) % n  # two members at least, where there is room
    if case["alone"]:
        group[B - case["alone"]:] = -1
    group = group[torch.randperm(B, generator=g)]
    shared = (case["prefix"] * (0.25 + 0.75 * torch.rand(n, generator=g)) / page).floor().long()
    shared[0] = case["prefix"] // page
    shared = shared.clamp(min=1)
    held = torch.where(group >= 0, shared[group.clamp(min=0)], torch.zeros_like(group)) * page
    keys = held + torch.randint(1, case["own_max"] + 1, (B,), generator=g)
    return group, shared, keys


def _prepare_attn(case, gen):
    B, page, Hq, Hkv = case["B"], case["page"], case["Hq"], case["Hkv"]
    group, shared, keys = _attn_shape(case)
    n_pages = (keys + page - 1) // page
    held = torch.where(group >= 0, shared[group.clamp(min=0)], torch.zeros_like(group))
    width = int(n_pages.max())
    total = int(shared.sum() + (n_pages - held).sum())
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(total))
    starts = torch.cumsum(shared, 0) - shared
    own_starts = int(shared.sum()) + torch.cumsum(n_pages - held, 0) - (n_pages - held)
    col = torch.arange(width)[None, :]
    index = torch.where(col < held[:, None], starts[group.clamp(min=0)][:, None] + col,
                        own_starts[:, None] + col - held[:, None])
    table = torch.where(col < n_pages[:, None], perm[index.clamp(0, total - 1)], torch.full_like(index, -1))
    i32 = dict(dtype=torch.int32, device="cuda")

    def normal(*s):
        return torch.empty(*s, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)

    cu = torch.zeros(B + 1, dtype=torch.int64)
    cu[1:] = torch.cumsum(keys, 0)
    return dict(q=normal(B, Hq, HD), k_cache=normal(total, page, Hkv, HD), v_cache=normal(total, page, Hkv, HD),
                cu_q=torch.arange(B + 1, **i32), cu_k=cu.to(**i32), max_k=int(keys.max()), table=table.to(**i32),
                group=group.to(**i32), prefix=(shared * page).to(**i32), scale=HD ** -0.5)


def _rows(case):
    """Lengths of all rows, from the case alone."""
    g = torch.Generator().manual_seed(613 * case["rows"] + 17 * case["max_len"] + case["pages"])
    return torch.randint(1, case["max_len"] + 1, (case["rows"],), generator=g).clamp(max=case["width"] * case["page"])


def _tables(case, lens, seed):
    """Tables with pages drawn without order, every sequence with its own."""
    page = case["page"]
    n_pages = (lens + page - 1) // page
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(case["pages"], generator=g)
    starts = torch.cumsum(n_pages, 0) - n_pages
    col = torch.arange(case["width"])[None, :]
    mine = col < n_pages[:, None]
    table = torch.where(mine, perm[(starts[:, None] + col).clamp(max=case["pages"] - 1)], torch.full((1, 1), -1))
    refs = torch.zeros(case["pages"], dtype=torch.int64)
    refs[table[mine]] = 1
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(table=table.to(**i32), lens=lens.to(**i32), refs=refs.to(**i32))


def _some(case, n, of, salt):
    g = torch.Generator().manual_seed(salt + 7 * n + of)
    return torch.randperm(of, generator=g)[:n]


def _fork_rows(case):
    """(parents, children): distinct children; several forks of one parent among them."""
    order = _some(case, case["rows"], case["rows"], 5)
    children, rest = order[:case["n"]], order[case["n"]:]
    return rest[torch.arange(case["n"]) % max(1, (rest.numel() + 1) // 2)], children


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "attn":
        return dict(case=case, **_prepare_attn(case, gen))
    i32 = dict(dtype=torch.int32, device="cuda")
    state = dict(case=case)
    if case["op"] != "turnover":
        state["kv"] = torch.empty(2, case["layers"], case["pages"], case["page"], case["Hkv"], HD,
                                  dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    if case["op"] == "copy":
        src, dst, tokens = _copy_pairs(case)
        return dict(state, src=src.to(**i32), dst=dst.to(**i32), tokens=None if tokens is None else tokens.to(**i32))
    lens = _rows(case)
    if case["op"] == "fork":
        parents, children = _fork_rows(case)
        return dict(state, parents=parents.to(**i32), children=children.to(**i32), **_tables(case, lens, seed))
    if case["op"] == "turnover":
        rows = _some(case, case["n"], case["rows"], 3)
        begin = _rows(dict(case, max_len=max(1, case["max_len"] - 1)))[rows]
        return dict(state, rows=rows.to(**i32), begin=begin.to(**i32), **_tables(case, lens, seed))
    lens = lens.clone()
    t = _tables(case, lens, seed)
    gone = _some(case, case["gone"], case["rows"], 11).cuda()
    pages = t["table"][gone]
    t["refs"][pages[pages >= 0].long()] = 0
    t["table"][gone] = -1
    t["lens"][gone] = 0
    return dict(state, **t, table0=t["table"].clone(), refs0=t["refs"].clone())


def _copy_pairs(case):
    order = _some(case, 2 * case["n"], case["pages"], 9)
    tokens = None
    if case["ragged"]:
        g = torch.Generator().manual_seed(case["n"] + case["pages"])
        tokens = torch.randint(0, case["page"] + 1, (case["n"],), generator=g)
    return order[:case["n"]], order[case["n"]:], tokens


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import os
    import sys
    pkg = os.path.join(os.getcwd(), "nano-vllm-diy_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from src import b200
    op = s["case"]["op"]
    if op == "attn":
        return b200.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["cu_k"], s["max_k"],
                                            s["scale"], s["table"], s["group"], s["prefix"])
    if op == "copy":
        b200.copy_pages(s["kv"], s["src"], s["dst"], s["tokens"])
        return s["kv"]
    if op == "fork":
        # a beam step: the children's rows are freed and taken by the forks (a second pass does the same)
        b200.free_pages(s["table"], s["lens"], s["refs"], s["children"])
        done = b200.fork_pages(s["kv"], s["table"], s["lens"], s["refs"], s["parents"], s["children"])
        return [s["kv"], s["table"], s["lens"], s["refs"], done]
    if op == "turnover":
        b200.free_pages(s["table"], s["lens"], s["refs"], s["rows"])
        done = b200.take_pages(s["table"], s["lens"], s["refs"], s["rows"], s["begin"], s["case"]["page"])
        return [s["table"], s["lens"], s["refs"], done]
    # the holes come back before each pass, so that every pass moves the same pages
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    moved = b200.compact_pages(s["kv"], s["table"], s["refs"])
    return [s["kv"], s["table"], s["refs"], moved]


def _plain_attn(s):
    B, Hq, _ = s["q"].shape
    page, Hkv = s["k_cache"].shape[1], s["k_cache"].shape[2]
    slots = s["table"].long().clamp(min=0)
    n = (s["cu_k"][1:] - s["cu_k"][:-1])[:, None, None, None]
    q = s["q"].float().view(B, Hkv, Hq // Hkv, HD) * s["scale"]
    k = s["k_cache"][slots].view(B, -1, Hkv, HD).permute(0, 2, 3, 1).float()
    scores = q @ k
    del k
    seen = torch.arange(scores.shape[-1], device=q.device)[None, None, None, :] < n
    scores = scores.masked_fill(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = s["v_cache"][slots].view(B, -1, Hkv, HD).permute(0, 2, 1, 3).float()
    return (p @ v).view(B, Hq, HD).to(torch.bfloat16)


def _plain_copy(kv, src, dst, tokens):
    """Pages dst := src (their first `tokens` slots) in every layer."""
    src, dst = src.long(), dst.long()
    if tokens is None:
        kv[:, :, dst] = kv[:, :, src]
        return
    head = torch.arange(kv.shape[3], device=kv.device)[None, :] < tokens[:, None]
    kv[:, :, dst] = torch.where(head[:, :, None, None], kv[:, :, src], kv[:, :, dst])


def _plain_free(table, lens, refs, rows):
    rows = rows.long()
    pages = table[rows]
    refs.index_add_(0, pages.clamp(min=0).flatten().long(), -(pages >= 0).flatten().to(torch.int32))
    table[rows] = -1
    lens[rows] = 0


def _plain_free_pages(refs):
    """(pages in the order free ones first, ascending; number of free ones)"""
    used = (refs > 0).to(torch.int32)
    return torch.argsort(used, stable=True), used.numel() - used.sum()


def _run_plain(s):
    op = s["case"]["op"]
    if op == "attn":
        return _plain_attn(s)
    if op == "copy":
        _plain_copy(s["kv"], s["src"], s["dst"], s["tokens"])
        return s["kv"]
    table, refs, page = s["table"], s["refs"], s["case"]["page"]
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    if op == "fork":
        lens, parents, children = s["lens"], s["parents"].long(), s["children"].long()
        _plain_free(table, lens, refs, children)
        n = lens[parents]
        full, part = n // page, n % page
        need = (part > 0).to(torch.int64)
        order, free = _plain_free_pages(refs)
        rank = torch.cumsum(need, 0)
        done = (need == 0) | (rank <= free)
        fresh = order[(rank - 1).clamp(0, order.numel() - 1)]
        has = done & (need > 0)
        old = table[parents]
        new = torch.where(col < full[:, None], old, torch.full_like(old, -1))
        new = torch.where((col == full[:, None]) & has[:, None], fresh[:, None].to(torch.int32), new)
        new = torch.where(done[:, None], new, torch.full_like(new, -1))
        last = old.gather(1, ((n + page - 1) // page - 1).clamp(min=0)[:, None].long())[:, 0].long()
        _plain_copy(s["kv"], last, torch.where(has, fresh, last), part)  # (no page of its own: the page onto itself)
        table[children] = new
        refs.index_add_(0, new.clamp(min=0).flatten().long(), (new >= 0).flatten().to(torch.int32))
        lens[children] = torch.where(done, n, torch.zeros_like(n))
        return [s["kv"], table, lens, refs, done.to(torch.int32)]
    if op == "turnover":
        lens, rows, begin = s["lens"], s["rows"].long(), s["begin"]
        _plain_free(table, lens, refs, rows)
        held = (lens[rows] + page - 1) // page
        need = (begin + page - 1) // page - held
        order, free = _plain_free_pages(refs)
        total = torch.cumsum(need, 0)
        done = total <= free
        index = (total - need - held)[:, None] + col
        fresh = (col >= held[:, None]) & (col < (held + need)[:, None]) & done[:, None]
        new = torch.where(fresh, order[index.clamp(0, order.numel() - 1).long()].to(torch.int32), table[rows])
        table[rows] = new
        refs.index_add_(0, new.clamp(min=0).flatten().long(), fresh.flatten().to(torch.int32))
        lens[rows] = torch.where(done, begin, lens[rows])
        return [table, lens, refs, done.to(torch.int32)]
    table.copy_(s["table0"])
    refs.copy_(s["refs0"])
    live = refs > 0
    n = live.sum()
    index = torch.arange(refs.numel(), device=refs.device)
    to = torch.nonzero(~live & (index < n))[:, 0]
    of = torch.nonzero(live & (index >= n))[:, 0]
    place = torch.where(live, index, torch.full_like(index, -1))
    place[of] = to
    _plain_copy(s["kv"], of, to, None)
    refs[to] = refs[of]
    refs[of] = 0
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()].to(torch.int32), table))
    return [s["kv"], table, refs, place.to(torch.int32)]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "attn":
        group, shared, keys = _attn_shape(case)
        of = torch.where(group >= 0, shared[group.clamp(min=0)] * case["page"], torch.zeros_like(group))
        used = shared[torch.unique(group[group >= 0])].sum() * case["page"]
        rows = int(used + (keys - of).sum())
        return {"bytes": rows * case["Hkv"] * HD * 4 + 2 * case["B"] * case["Hq"] * HD * 2,
                "flops": 4 * HD * case["Hq"] * int(keys.sum())}
    slot = 2 * case.get("layers", 0) * case.get("Hkv", 0) * HD * 2  # bytes of one token in every layer
    if case["op"] == "copy":
        tokens = _copy_pairs(case)[2]
        return {"bytes": 2 * slot * (case["n"] * case["page"] if tokens is None else int(tokens.sum())), "flops": 0}
    lens = _rows(case)
    page = case["page"]
    if case["op"] == "turnover":
        rows = _some(case, case["n"], case["rows"], 3)
        begin = _rows(dict(case, max_len=max(1, case["max_len"] - 1)))[rows]
        pages = int(((lens[rows] + page - 1) // page).sum() + ((begin + page - 1) // page).sum())
        return {"bytes": 4 * (case["pages"] + 4 * pages + 4 * case["n"]), "flops": 0}
    if case["op"] == "fork":
        parents, children = _fork_rows(case)
        pages = int(((lens[parents] + page - 1) // page).sum() + ((lens[children] + page - 1) // page).sum())
        return {"bytes": 2 * slot * int((lens[parents] % page).sum()) + 4 * (case["pages"] + 4 * pages), "flops": 0}
    n_pages = (lens + page - 1) // page
    gone = _some(case, case["gone"], case["rows"], 11)
    live = int(n_pages.sum() - n_pages[gone].sum())
    # the pages lie at random: of `live` ones the share (pages - live) / pages is behind the first `live` places
    moved = live * (case["pages"] - live) / case["pages"]
    return {"bytes": 2 * slot * page * moved + 8 * case["rows"] * case["width"] + 8 * case["pages"], "flops": 0}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        cu, table, page = s["cu_k"].tolist(), s["table"].tolist(), case["page"]
        for b in range(case["B"]):
            n = cu[b + 1] - cu[b]
            pages = table[b][:-(-n // page)]
            k = s["k_cache"][pages].flatten(0, 1)[:n].double().repeat_interleave(case["Hq"] // case["Hkv"], 1)
            v = s["v_cache"][pages].flatten(0, 1)[:n].double().repeat_interleave(case["Hq"] // case["Hkv"], 1)
            w = torch.softmax(torch.einsum("hd,nhd->hn", s["q"][b].double(), k) * s["scale"], -1)
            out[b] = torch.einsum("hn,nhd->hd", w, v)
        return out
    kv = s.get("kv")
    if case["op"] == "copy":
        tokens = [case["page"]] * case["n"] if s["tokens"] is None else s["tokens"].tolist()
        for a, b, t in zip(s["src"].tolist(), s["dst"].tolist(), tokens):
            kv[:, :, b, :t] = kv[:, :, a, :t]
        return kv
    table, refs, page = s["table"].tolist(), s["refs"].tolist(), case["page"]
    if case["op"] == "compact":
        n = sum(r > 0 for r in refs)
        holes = [p for p in range(n) if refs[p] == 0]
        place = [p if r > 0 else -1 for p, r in enumerate(refs)]
        for p in range(n, len(refs)):
            if refs[p] > 0:
                to = holes.pop(0)
                kv[:, :, to] = kv[:, :, p]
                place[p], refs[to], refs[p] = to, refs[p], 0
        table = [[place[e] if e >= 0 else -1 for e in row] for row in table]
        return [kv, torch.tensor(table), torch.tensor(refs), torch.tensor(place)]
    lens = s["lens"].tolist()

    def leave(rows):
        for r in rows:
            for e in table[r]:
                if e >= 0:
                    refs[e] -= 1
            table[r], lens[r] = [-1] * case["width"], 0

    free = None
    done = []
    if case["op"] == "turnover":
        leave(s["rows"].tolist())
        free = [p for p, r in enumerate(refs) if r == 0]
        asked = 0
        for r, n in zip(s["rows"].tolist(), s["begin"].tolist()):
            need = -(-n // page)
            asked += need
            done.append(int(asked <= len(free)))
            if done[-1]:
                for j, p in enumerate(free[asked - need:asked]):
                    table[r][j], refs[p] = p, 1
                lens[r] = n
        return [torch.tensor(table), torch.tensor(lens), torch.tensor(refs), torch.tensor(done)]
    leave(s["children"].tolist())
    free = [p for p, r in enumerate(refs) if r == 0]
    for a, c in zip(s["parents"].tolist(), s["children"].tolist()):
        n = lens[a]
        full, part = divmod(n, page)
        done.append(int(part == 0 or len(free) > 0))
        if not done[-1]:
            continue
        table[c][:full] = table[a][:full]
        for e in table[a][:full]:
            refs[e] += 1
        if part:
            p = free.pop(0)
            kv[:, :, p, :part] = kv[:, :, table[a][full], :part]
            table[c][full], refs[p] = p, 1
        lens[c] = n
    return [kv, torch.tensor(table), torch.tensor(lens), torch.tensor(refs), torch.tensor(done)]
