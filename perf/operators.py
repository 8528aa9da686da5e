"""The serving operators over the paged pool, as cases that can be timed: the step's tables, the rows' way into the pool with
the blocks' mean keys, and attention over the blocks that a cheap score selects.

`own` false: the operators from elementary torch operations; `own` true: the calls a user makes of `silvann_b200.ext`.
"""
import math

import torch

own = False

FP16, BF16 = 0, 1
_TYPES = {FP16: torch.float16, BF16: torch.bfloat16}
_LOWEST = -1e308      # what a score that is no number, or minus infinity, ranks as: above what is no candidate at all


def listed():
    return [
        # --- the step's tables: which pages and slots this step's new positions get ---
        # an ordinary decode step: every sequence of the 32-sequence batch gets one more position
        {"name": "tables decode 32", "op": "tables", "seqs": 32, "lo": 1024, "hi": 100000, "c_lo": 1, "c_hi": 1, "ended": 0, "page": 256, "pad": 0},
        # a large batch in flight: some sequences end (their pages come back), some wait, the rest get one position, with
        # room in the row arrays for more (a captured step's fixed capacity)
        {"name": "tables decode 4097", "op": "tables", "seqs": 4097, "lo": 1, "hi": 2000, "c_lo": 0, "c_hi": 1, "ended": 16, "page": 64, "pad": 511},
        # prompts enter: 61 sequences of very different lengths bring 98 thousand new positions
        {"name": "tables prompts 61", "op": "tables", "seqs": 61, "lo": 0, "hi": 3000, "c_lo": 1, "c_hi": 3201, "ended": 0, "page": 16, "pad": 7},
        # --- rows into the pool ---
        # a decode step's rows: one a sequence, 2 kv heads of 256; a row in sixty-four completes a block
        {"name": "write decode 32", "op": "write", "seqs": 32, "lo": 1024, "hi": 9000, "c_lo": 1, "c_hi": 1, "kv_heads": 2, "head_dim": 256, "dtype": BF16, "page": 256, "block": 64, "gap": 0, "pad": 0},
        # a prompt chunk of a few sequences out of a fused projection (the rows are wider than the keys), small blocks
        {"name": "write chunk 4 of 2000", "op": "write", "seqs": 4, "lo": 0, "hi": 777, "c_lo": 1800, "c_hi": 2201, "kv_heads": 4, "head_dim": 128, "dtype": FP16, "page": 64, "block": 16, "gap": 2048, "pad": 33},
        # the largest: a batch of whole prompts
        {"name": "write prompts 64", "op": "write", "seqs": 64, "lo": 0, "hi": 500, "c_lo": 200, "c_hi": 2100, "kv_heads": 2, "head_dim": 256, "dtype": BF16, "page": 256, "block": 64, "gap": 0, "pad": 0},
        # --- attention over selected blocks ---
        # short sequences whose every block is kept: the floor of a call
        {"name": "sparse short 7", "op": "sparse", "seqs": 7, "lo": 1, "hi": 300, "drafts": 1, "q_heads": 24, "kv_heads": 2, "head_dim": 64, "dtype": FP16, "page": 64, "block": 32, "first": 1, "last": 2, "top": 13},
        # one sequence of 8,192 positions, 16 query heads on 4 kv heads of 128: one user's decode step
        {"name": "sparse one 8192", "op": "sparse", "seqs": 1, "lo": 8192, "hi": 8192, "drafts": 1, "q_heads": 16, "kv_heads": 4, "head_dim": 128, "dtype": FP16, "page": 256, "block": 64, "first": 1, "last": 2, "top": 13},
        # one long context: 262,144 positions, 32 query heads on 4 kv heads of 128
        {"name": "sparse one 262144", "op": "sparse", "seqs": 1, "lo": 262144, "hi": 262144, "drafts": 1, "q_heads": 32, "kv_heads": 4, "head_dim": 128, "dtype": BF16, "page": 256, "block": 64, "first": 1, "last": 4, "top": 59},
        # several drafted positions a sequence, a kv head for every query head, small pages
        {"name": "sparse drafts 24x5", "op": "sparse", "seqs": 24, "lo": 500, "hi": 20000, "drafts": 5, "q_heads": 8, "kv_heads": 8, "head_dim": 64, "dtype": FP16, "page": 16, "block": 16, "first": 2, "last": 4, "top": 26},
        # the ragged batch of 32 sequences of 1,024 to 100,000 positions, 16 query heads on 2 kv heads of 256
        {"name": "sparse batch 32", "op": "sparse", "seqs": 32, "lo": 1024, "hi": 100000, "drafts": 1, "q_heads": 16, "kv_heads": 2, "head_dim": 256, "dtype": BF16, "page": 256, "block": 64, "first": 1, "last": 2, "top": 29},
        # the largest: a full server
        {"name": "sparse batch 256", "op": "sparse", "seqs": 256, "lo": 1000, "hi": 16000, "drafts": 1, "q_heads": 32, "kv_heads": 4, "head_dim": 128, "dtype": BF16, "page": 128, "block": 128, "first": 1, "last": 1, "top": 14},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "write", "sparse", "sparse"])
    if op == "tables":
        seqs = _spread(rng, 1, 6000)
        c_hi = _spread(rng, 1, max(1, min(3000, 90000 // seqs)))
        return {"op": op, "seqs": seqs, "lo": 0, "hi": _spread(rng, 1, max(2, min(60000, 2000000 // seqs))), "c_lo": rng.choice([0, 1]), "c_hi": c_hi,
                "ended": rng.choice([0, 0, 3, 10, 50]), "page": rng.choice([16, 32, 48, 64, 128, 256]), "pad": rng.randrange(0, 300)}
    block = rng.choice([16, 32, 64, 128])
    page = block * rng.choice([1, 1, 2, 3, 4])
    dtype = rng.choice([FP16, BF16])
    if op == "write":
        seqs = _spread(rng, 1, 200)
        kv_heads, head_dim = rng.choice([(1, 64), (2, 64), (8, 64), (1, 128), (4, 128), (8, 128), (2, 256), (4, 256)])
        most = 60000 * 512 // (kv_heads * head_dim)
        c_hi = _spread(rng, 1, max(1, min(4000, most // seqs)))
        return {"op": op, "seqs": seqs, "lo": 0, "hi": _spread(rng, 1, 700), "c_lo": rng.choice([1, (c_hi + 1) // 2, c_hi]), "c_hi": c_hi, "kv_heads": kv_heads, "head_dim": head_dim,
                "dtype": dtype, "page": page, "block": block, "gap": rng.choice([0, 0, 8, 4 * head_dim]), "pad": rng.randrange(0, 40)}
    head_dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8, 12, 16])
    seqs = _spread(rng, 1, 160)
    drafts = rng.choice([1, 1, 1, 2, 4])
    keep = _spread(rng, 4, max(5, min(64, 2048 // block)))
    first, last = rng.choice([0, 1, 2]), rng.choice([1, 2])
    # a drawn case gathers no more than the largest listed one
    seqs = max(1, min(seqs, 256 * 4 * 128 * 2048 // (drafts * kv_heads * head_dim * keep * block)))
    hi = _spread(rng, 50, max(60, min(200000, 100000000 // (seqs * kv_heads * head_dim))))
    return {"op": op, "seqs": seqs, "lo": max(drafts, hi // rng.choice([1, 2, 10, 100])), "hi": max(drafts, hi), "drafts": drafts, "q_heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "page": page, "block": block, "first": first, "last": last, "top": keep - first - last}


def _between(n, lo, hi, turn):
    """n whole numbers spread evenly over lo..hi, in an order without a pattern: the case's own, whatever the seed."""
    return [lo + int((hi - lo + 1) * ((0.5 + i * 0.6180339887498949 + turn) % 1.0)) for i in range(n)]


def _lengths(case):
    """(lens, counts) of a case: positions held before the step, new ones (-1: the sequence has ended)."""
    lens = _between(case["seqs"], case["lo"], case["hi"], 0.0)
    if case["op"] == "sparse":
        return lens, None
    counts = _between(case["seqs"], case["c_lo"], case["c_hi"], 0.37)
    every = case.get("ended", 0)
    if every:
        counts = [-1 if i % every == every // 2 else c for i, c in enumerate(counts)]
    return lens, counts


def _pages(n, page):
    return (n + page - 1) // page


def _tables(lens, need, page, g):
    """Random distinct pages for every sequence's first `lens` positions: (page table [seqs][stride], pages in all, a random
    order of all pages whose first ones are those in use).  `need`: the columns a row has."""
    held = torch.tensor([_pages(n, page) for n in lens])
    total, stride = int(held.sum()), max(1, max(need))
    spare = sum(need) - total
    order = torch.randperm(total + spare, generator=g, device="cuda").int()
    start = torch.cumsum(held, 0) - held
    col = torch.arange(stride)
    inside = (col[None] < held[:, None]).cuda()
    at = (start[:, None] + col[None]).clamp_(max=total + spare - 1).cuda()
    return torch.where(inside, order[at], -1).int().contiguous(), total + spare, order, total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, counts = _lengths(case)
    page = case["page"]
    st = dict(case)
    if case["op"] == "tables":
        now = [max(0, c) + n for n, c in zip(lens, counts)]
        table, pool_pages, free, used = _tables(lens, [_pages(n, page) for n in now], page, g)
        # the seed turns which sequence has which length
        turn = torch.randperm(case["seqs"], generator=g, device="cuda")
        rows = sum(c for c in counts if c > 0) + case["pad"]
        i32 = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")  # noqa: E731
        st.update(lens=torch.tensor(lens, dtype=torch.int32, device="cuda")[turn].contiguous(), counts=torch.tensor(counts, dtype=torch.int32, device="cuda")[turn].contiguous(),
                  table=table[turn].contiguous(), free=free.contiguous(), free_at=torch.tensor([used], dtype=torch.int32, device="cuda"), pool_pages=pool_pages, rows=max(1, rows),
                  stride=table.shape[1], new_lens=i32(case["seqs"]), free_out=i32(1), row_start=i32(case["seqs"] + 1), row_seq=i32(max(1, rows)), row_pos=i32(max(1, rows)),
                  row_slot=i32(max(1, rows)))
        return st
    kvh, d, block, dt = case["kv_heads"], case["head_dim"], case["block"], _TYPES[case["dtype"]]
    now = lens if counts is None else [n + c for n, c in zip(lens, counts)]
    table, pool_pages, _, _ = _tables(now, [_pages(n, page) for n in now], page, g)
    new = torch.tensor([case["drafts"]] * case["seqs"] if counts is None else counts)
    seq = torch.repeat_interleave(new)
    pos = (torch.tensor(now) - torch.cumsum(new, 0))[seq] + torch.arange(seq.numel())
    seq, pos = seq.int().cuda(), pos.int().cuda()
    # keys share a direction within a block, as neighbouring positions do; one page more than the pool has is behind it
    blocks = (pool_pages + 1) * (page // block)
    k = torch.randn((blocks, block, kvh, d), generator=g, device="cuda", dtype=dt)
    k += torch.randn((blocks, 1, kvh, d), generator=g, device="cuda", dtype=dt) * 0.5
    v = torch.randn((pool_pages + 1, page, kvh, d), generator=g, device="cuda", dtype=dt)
    k = k.view(pool_pages + 1, page, kvh, d)
    means = torch.cat([b.float().mean(1).to(dt) for b in k.view(blocks, block, kvh, d).split(8192)])
    st.update(k_all=k, v_all=v, means=means.view(pool_pages + 1, page // block, kvh, d), table=table, pool_pages=pool_pages, stride=table.shape[1])
    if case["op"] == "write":
        slot = table[seq.long(), (pos // page).long()] * page + pos % page
        pad = torch.full((case["pad"],), -1, dtype=torch.int32, device="cuda")
        slot = torch.cat([slot, pad]).int().contiguous()
        wide = torch.randn((slot.numel(), 2 * kvh * d + case["gap"]), generator=g, device="cuda", dtype=dt)
        st.update(slot=slot, rows=slot.numel(), wide=wide, k_rows=wide[:, :kvh * d], v_rows=wide[:, kvh * d:2 * kvh * d], row_stride=wide.shape[1])
        return st
    rows, keep = seq.numel(), case["first"] + case["last"] + case["top"]
    q = torch.randn((rows, case["q_heads"], d), generator=g, device="cuda", dtype=dt)
    st.update(q=q, seq=seq, pos=pos, rows=rows, keep=keep, blocks=(max(now) - 1) // block + 1, o=torch.empty_like(q),
              chosen=torch.empty((rows, kvh, keep), dtype=torch.int32, device="cuda"))
    return st


def run(state):
    return {"tables": _run_tables, "write": _run_write, "sparse": _run_sparse}[state["op"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _run_tables(s):
    page, stride = s["page"], s["stride"]
    if own:
        from silvann_b200 import ext
        ext.paged_tables(s["new_lens"], s["table"], s["row_start"], s["row_seq"], s["row_pos"], s["row_slot"], s["free_out"], s["free"], s["free_at"], s["lens"], s["counts"], s["seqs"],
                         stride, s["rows"], s["free"].numel(), s["pool_pages"], page, stream=_stream())
        return {"lens": s["new_lens"], "table": s["table"], "start": s["row_start"], "seq": s["row_seq"], "pos": s["row_pos"], "slot": s["row_slot"], "free_at": s["free_out"], "free": s["free"]}
    lens, counts = s["lens"].long(), s["counts"].long()
    gone = counts < 0
    new = torch.where(gone, 0, lens + counts)
    held = (lens + page - 1) // page
    need = torch.where(gone, 0, (new + page - 1) // page - held)
    back = torch.where(gone, held, 0)
    start = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.cumsum(counts.clamp(min=0), 0)])
    bottom = s["free_at"].long() - back.sum()
    col = torch.arange(stride, device="cuda")
    # pages that come back, in order, below the free ones; then the pages handed out from the bottom of what is free now
    n_free = s["free"].numel()
    to = torch.where(col[None] < back[:, None], bottom + (torch.cumsum(back, 0) - back)[:, None] + col[None], n_free)
    free = torch.cat([s["free"], s["free"][:1]]).index_put((to.reshape(-1),), s["table"].reshape(-1))[:n_free].contiguous()
    taken = col[None] - held[:, None]
    frm = (bottom + (torch.cumsum(need, 0) - need)[:, None] + taken).clamp(0, n_free - 1)
    table = torch.where((taken >= 0) & (taken < need[:, None]), free[frm], s["table"])
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(start[1:], r, right=True).clamp(max=s["seqs"] - 1)
    inside = r < start[-1]
    pos = lens[seq] + r - start[seq]
    slot = table[seq, (pos // page).clamp(0, stride - 1)].long() * page + pos % page
    pad = lambda x: torch.where(inside, x, -1).int()  # noqa: E731
    return {"lens": new.int(), "table": table, "start": start.int(), "seq": pad(seq), "pos": pad(pos), "slot": pad(slot), "free_at": (bottom + need.sum()).int(), "free": free}


def _run_write(s):
    kvh, d, page, block, pages = s["kv_heads"], s["head_dim"], s["page"], s["block"], s["pool_pages"]
    k, v, means = s["k_all"], s["v_all"], s["means"]
    if own:
        from silvann_b200 import ext
        ext.paged_write(k, v, means, s["k_rows"], s["v_rows"], s["slot"], s["rows"], kvh, d, pages, page, block, k_stride=s["row_stride"], v_stride=s["row_stride"], dtype=s["dtype"], stream=_stream())
        return {"k": k[:pages], "v": v[:pages], "means": means[:pages]}
    behind = pages * page
    slot = torch.where(s["slot"] < 0, behind, s["slot"]).long()
    k.view(-1, kvh * d).index_copy_(0, slot, s["k_rows"])
    v.view(-1, kvh * d).index_copy_(0, slot, s["v_rows"])
    # the rows that complete a block, first: there are at most one in `block` and one a sequence
    done = (s["slot"] >= 0) & (slot % block == block - 1)
    done, at = torch.sort(done, descending=True, stable=True)
    most = min(s["rows"], s["rows"] // block + s["seqs"])
    whole = torch.where(done[:most], slot[at[:most]] // block, means.shape[0] * means.shape[1] - 1)
    means.view(-1, kvh, d).index_copy_(0, whole, k.view(-1, block, kvh, d)[whole].float().mean(1).to(k.dtype))
    return {"k": k[:pages], "v": v[:pages], "means": means[:pages]}


def _run_sparse(s):
    kvh, d, page, block, keep = s["kv_heads"], s["head_dim"], s["page"], s["block"], s["keep"]
    if own:
        from silvann_b200 import ext
        ext.paged_sparse(s["o"], None, s["chosen"], s["q"], s["k_all"], s["v_all"], s["means"], s["seq"], s["pos"], s["rows"], s["table"], s["seqs"], s["stride"], s["pool_pages"], page, block,
                         s["q_heads"], kvh, d, s["first"], s["last"], s["top"], dtype=s["dtype"], stream=_stream())
        return {"o": s["o"], "chosen": s["chosen"]}
    rows, group, per = s["rows"], s["q_heads"] // kvh, page // block
    seq, pos = s["seq"].long(), s["pos"].long()
    q = s["q"].view(rows, kvh, group, d)
    n = pos // block + 1
    # the cheap score, in 64 bits: the choice hangs on values next to a border
    j = torch.arange(s["blocks"], device="cuda")
    at = s["table"][seq[:, None], (j // per)[None]].clamp(min=0).long() * per + (j % per)[None]
    score = torch.einsum("rgd,rjgd->rgj", q.double().sum(2), s["means"].view(-1, kvh, d)[at].double())
    score = torch.where(score > _LOWEST, score, _LOWEST)
    middle = (n[:, None] > keep) & (j[None] >= s["first"]) & (j[None] < n[:, None] - s["last"])
    score = torch.where(middle[:, None], score, -math.inf)
    order = torch.sort(score, dim=2, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, j.expand_as(order))
    taken = (j[None] < n[:, None]) & ~middle
    taken = taken[:, None] | (middle[:, None] & (rank < s["top"]))
    ids = torch.where(taken, j, s["blocks"]).sort(dim=2).values
    ids = torch.nn.functional.pad(ids, (0, max(0, keep - s["blocks"])), value=s["blocks"])[:, :, :keep]
    ids = torch.where(ids < s["blocks"], ids, -1)
    # attention over the chosen blocks' positions up to the row's own
    p = (ids[..., None] * block + torch.arange(block, device="cuda")).view(rows, kvh, keep * block)
    inside = (p >= 0) & (p <= pos[:, None, None])
    p = p.clamp(min=0)
    slot = s["table"][seq[:, None, None], (p // page).clamp(max=s["stride"] - 1)].clamp(min=0).long() * page + p % page
    head = torch.arange(kvh, device="cuda")[None, :, None]
    w = torch.einsum("rgad,rgld->rgal", q.float(), s["k_all"].view(-1, kvh, d)[slot, head].float()) / math.sqrt(d)
    w = torch.where(inside[:, :, None], w, -math.inf)
    w = torch.exp(w - w.amax(3, keepdim=True))
    v = torch.where(inside[..., None], s["v_all"].view(-1, kvh, d)[slot, head].float(), 0.0)
    o = torch.einsum("rgal,rgld->rgad", w, v) / w.sum(3, keepdim=True)
    return {"o": o.reshape(rows, s["q_heads"], d).to(s["q"].dtype), "chosen": ids.int()}


def work(case):
    lens, counts = _lengths(case)
    page = case["page"]
    if case["op"] == "tables":
        rows, old, new = sum(c for c in counts if c > 0), sum(_pages(n, page) for n, c in zip(lens, counts) if c < 0), sum(_pages(n + c, page) - _pages(n, page) for n, c in zip(lens, counts) if c >= 0)
        return {"bytes": 16 * case["seqs"] + 12 * (rows + case["pad"]) + 8 * (old + new), "flops": 0}
    kvh, d, block = case["kv_heads"], case["head_dim"], case["block"]
    if case["op"] == "write":
        rows, whole = sum(counts), sum((n + c) // block - n // block for n, c in zip(lens, counts))
        before = sum(n % block for n, c in zip(lens, counts) if (n + c) // block > n // block)     # rows of earlier steps in a block that this one completes
        return {"bytes": (4 * rows + before + whole) * kvh * d * 2 + 4 * (rows + case["pad"]), "flops": (whole * block) * kvh * d}
    keep, group = case["first"] + case["last"] + case["top"], case["q_heads"] // kvh
    bytes_, flops = 0, 0
    for n in lens:
        blocks = (n - 1) // block + 1
        if blocks > keep:
            bytes_ += (blocks - case["first"] - case["last"]) * kvh * d * 2
            flops += case["drafts"] * 2 * (blocks - case["first"] - case["last"]) * kvh * d
        at = min(n, (keep - 1) * block + (n - 1) % block + 1)
        bytes_ += min(n, at * case["drafts"]) * kvh * d * 4
        flops += case["drafts"] * at * kvh * group * d * 4
    rows = len(lens) * case["drafts"]
    return {"bytes": bytes_ + rows * (case["q_heads"] * d * 4 + kvh * keep * 4 + 8), "flops": flops}


def exact(case, seed):
    if case["op"] == "tables":
        return None          # whole numbers: nothing is computed
    s = prepare(case, seed)
    kvh, d, page, block = case["kv_heads"], case["head_dim"], case["page"], case["block"]
    if case["op"] == "write":
        pages = s["pool_pages"]
        k, v, m = (x.double().reshape(-1, kvh, d) for x in (s["k_all"], s["v_all"], s["means"]))
        here = torch.nonzero(s["slot"] >= 0).reshape(-1)
        slot = s["slot"][here].long()
        k[slot] = s["k_rows"][here].double().view(-1, kvh, d)
        v[slot] = s["v_rows"][here].double().view(-1, kvh, d)
        done = slot[(slot + 1) % block == 0] // block
        m[done] = torch.stack([k[done * block + i] for i in range(block)]).sum(0) / block
        shape = (pages + 1, page, kvh, d)
        return {"k": k.view(shape)[:pages], "v": v.view(shape)[:pages], "means": m.view(pages + 1, -1, kvh, d)[:pages]}
    group, first, last, top = case["q_heads"] // kvh, case["first"], case["last"], case["top"]
    kp, vp, mp = (s[x].view(-1, kvh, d) for x in ("k_all", "v_all", "means"))
    out, ids = torch.zeros((s["rows"], kvh, group, d), dtype=torch.float64, device="cuda"), torch.full((s["rows"], kvh, s["keep"]), -1, dtype=torch.int32)
    lanes = torch.arange(block, device="cuda")
    for r, (seq, p) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
        pages = s["table"][seq, :p // page + 1].long()
        n = p // block + 1
        starts = (pages[:, None] * page + torch.arange(0, page, block, device="cuda")).reshape(-1)[:n]      # each block's first slot
        q = s["q"][r].double().view(kvh, group, d)
        pick = torch.arange(n, device="cuda").expand(kvh, n)
        if n > s["keep"]:
            sc = (mp[starts[first:n - last] // block].double() * q.sum(1)).sum(2).T
            best = torch.sort(sc.nan_to_num(nan=-math.inf), dim=1, descending=True, stable=True).indices[:, :top] + first
            ends = torch.cat([torch.arange(first, device="cuda"), torch.arange(n - last, n, device="cuda")]).expand(kvh, first + last)
            pick = torch.cat([best, ends], 1).sort(dim=1).values
        ids[r, :, :pick.shape[1]] = pick.int().cpu()
        slots = (starts[pick][..., None] + lanes).flatten(1)[:, :(pick.shape[1] - 1) * block + p % block + 1]
        heads = torch.arange(kvh, device="cuda")[:, None]
        w = torch.softmax(q @ kp[slots, heads].double().transpose(1, 2) / math.sqrt(d), 2)
        out[r] = w @ vp[slots, heads].double()
    return {"o": out.view(s["rows"], case["q_heads"], d), "chosen": ids.cuda()}
