"""The operators of a decode step that adds several rows to each sequence, as measured cases.

A step that verifies drafted tokens, or that takes a prompt chunk of each of several
sequences, runs four operators over the paged KV cache:

  plan    page tables, row starts, positions and cache slots from the sequences' lengths (b2_kv_plan)
  append  RoPE of the new rows' q and k, k and v into their cache slots (b2_rows_append)
  attn    attention of the new rows over cache and tree, or cache and earlier rows (b2_attn_rows)
  accept  the greedily accepted branch of each tree, its K/V moved together in every layer
          (b2_tree_accept, b2_kv_compact)

`own` False computes them with elementary torch operations, True with the library.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64  # tokens of a page in the library's own contexts

# head layouts of this repository's workloads: the 8B shape, the small GQA decoder, the tiny q8
# decoder, and one rank of the 70B shape on eight GPUs
SHAPES = {"8b": (32, 8, 128), "small": (9, 3, 64), "tiny": (6, 6, 48), "70b_rank": (8, 1, 128)}


def _attn(name, shape, batch, tokens, ctx, tree, page=PAGE):
    h, hkv, hd = SHAPES[shape]
    return {"name": name, "op": "attn", "heads": h, "kv_heads": hkv, "head_dim": hd, "batch": batch, "tokens": tokens,
            "ctx": ctx, "tree": tree, "page": page}


def listed():
    return [
        # one user, eight drafted tokens, a short conversation: latency
        _attn("attn 8b tree 8 ctx 1000", "8b", 1, 8, 1000, True),
        # one user of the tiny decoder, pages of 16
        _attn("attn tiny tree 5 ctx 141", "tiny", 1, 5, 141, True, 16),
        # a batch of the small GQA decoder near its context limit
        _attn("attn small b16 tree 16", "small", 16, 16, 2000, True),
        # a serving batch at the 8B shape with wide trees and ragged contexts
        _attn("attn 8b b16 tree 32 ctx 8000", "8b", 16, 32, 8000, True),
        # long contexts, a rank of the 70B shape
        _attn("attn 70b rank b8 ctx 30000", "70b_rank", 8, 16, 30000, True),
        # a prompt chunk deep in a context
        _attn("attn 8b chunk 512 ctx 2500", "8b", 1, 512, 2500, False),
        # a handful of trees
        {"name": "plan b4 tree", "op": "plan", "batch": 4, "tokens": 24, "ctx": 700, "tree": True, "page": PAGE},
        # many requests, prompt chunks among them
        {"name": "plan b1024 chunks", "op": "plan", "batch": 1024, "tokens": 256, "ctx": 6000, "tree": False, "page": PAGE},
        # one small tree, and a batch of prompt chunks
        {"name": "append 8b rows 8", "op": "append", "heads": 32, "kv_heads": 8, "head_dim": 128, "rows": 8, "page": PAGE},
        {"name": "append 8b rows 2048", "op": "append", "heads": 32, "kv_heads": 8, "head_dim": 128, "rows": 2048, "page": PAGE},
        # one user of the small decoder (30 layers), and a serving batch at the 8B shape (32 layers)
        {"name": "accept small b1", "op": "accept", "kv_heads": 3, "head_dim": 64, "layers": 30, "batch": 1, "tokens": 8,
         "keep": 4, "ctx": 500, "page": PAGE},
        {"name": "accept 8b b16", "op": "accept", "kv_heads": 8, "head_dim": 128, "layers": 32, "batch": 16, "tokens": 32,
         "keep": 6, "ctx": 90, "page": PAGE},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "plan", "append", "accept"])
    page = rng.choice([16, 24, 64, 64, 64, 128])
    hkv = rng.choice([1, 2, 3, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    hd = rng.choice([48, 64, 80, 128, 128])
    if op == "attn":
        tree = rng.random() < 0.7
        batch = _log(rng, 1, 16) if tree else _log(rng, 1, 4)
        tokens = rng.randint(1, 64) if tree else _log(rng, 1, 500)
        # queries times keys no more than the largest listed case's
        most = min(30000, int(3.0e9 / (batch * hkv * group * tokens * hd)), int(4.0e7 / (batch * hkv)))
        return {"op": op, "heads": hkv * group, "kv_heads": hkv, "head_dim": hd, "batch": batch, "tokens": tokens,
                "ctx": _log(rng, 1, max(2, most)), "tree": tree, "page": page}
    if op == "plan":
        tree = rng.random() < 0.5
        return {"op": op, "batch": _log(rng, 1, 1000), "tokens": rng.randint(1, 64) if tree else _log(rng, 1, 250),
                "ctx": _log(rng, 1, 6000), "tree": tree, "page": page}
    if op == "append":
        return {"op": op, "heads": hkv * group, "kv_heads": hkv, "head_dim": hd, "rows": _log(rng, 1, 1000), "page": page}
    tokens = rng.randint(2, 64)
    return {"op": op, "kv_heads": hkv, "head_dim": hd, "layers": rng.randint(1, 16), "batch": _log(rng, 1, 16),
            "tokens": tokens, "keep": rng.randint(1, min(8, tokens)), "ctx": _log(rng, 1, 90), "page": page}


# ---- inputs ---------------------------------------------------------------------------------------


def _lengths(case):
    """Cached and new lengths of each sequence, a case's own: the first has the case's, the rest are ragged up to them."""
    b = case["batch"]
    rng = np.random.default_rng([b, case["tokens"], case["ctx"]])
    ctx = rng.integers(case["ctx"] // 2, case["ctx"] + 1, b)
    new = rng.integers((case["tokens"] + 1) // 2, case["tokens"] + 1, b)
    ctx[0], new[0] = case["ctx"], case["tokens"]
    return ctx.astype(np.int64), new.astype(np.int64)


def _parents(n, rng):
    """A drafted tree in topological order: node 0 is the token just decoded; most nodes extend a recent one."""
    return [-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)]


def _masks(parents):
    m = []
    for i, p in enumerate(parents):
        m.append((m[p] if p >= 0 else 0) | (1 << i))
    return m


def _signed(masks):
    return torch.from_numpy(np.array(masks, np.uint64).view(np.int64)).cuda()


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _tables(total, page, rng, slack=0):
    """Shuffled pages: table rows [b][pages], the pages in use of each sequence, the free pages, and the pool's size."""
    used = -(-total // page)
    pps = int(used.max()) + slack
    n = int(used.sum()) + 8 + slack * len(total)
    order = rng.permutation(n)
    table = np.full((len(total), pps), -1, np.int64)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    return table, used, order[at:], n


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op, page = case["op"], case["page"]
    st = {"case": case, "op": op, "page": page}
    if op == "append":
        h, hkv, hd, rows = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
        pages = -(-rows // page) + 4
        st["y"] = normal(rows, (h + 2 * hkv) * hd)
        st["positions"] = _i32(rng.integers(0, 8000, rows))
        st["slots"] = _i32(rng.permutation(pages * page)[:rows])
        st["freq"] = (1.0 / 500000.0 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)).float()
        st["q"] = torch.zeros(rows, h * hd, device="cuda")
        st["k"], st["v"] = normal(pages, hkv, page, hd), normal(pages, hkv, page, hd)
        st["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return st
    ctx, new = _lengths(case)
    b, rows = case["batch"], int(new.sum())
    start = np.concatenate([[0], np.cumsum(new)])
    st["rows"], st["longest"], st["most_new"] = rows, int((ctx + new).max()), int(new.max())
    st["ctx_len"], st["new_len"] = _i32(ctx), _i32(new)
    st["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    parents = [_parents(int(n), rng) for n in new] if case.get("tree") or op == "accept" else None
    st["tree"] = _signed([m for p in parents for m in _masks(p)]) if parents else None
    if op == "plan":
        have = -(-ctx // page)
        table, used, free, n = _tables(ctx, page, rng, slack=-(-case["tokens"] // page) + 1)
        st.update(table=_i32(table), mapped=_i32(have), free=_i32(free), free_count=_i32([len(free)]), pool_pages=n)
        st.update(mapped_out=torch.zeros_like(st["mapped"]), free_out=torch.zeros_like(st["free_count"]),
                  row_start=torch.zeros(b + 1, dtype=torch.int32, device="cuda"))
        for k in ("row_item", "row_pos", "row_slot"):
            st[k] = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
        return st
    st["row_start"] = _i32(start)
    st["row_item"] = _i32(np.repeat(np.arange(b), new))
    st["row_local"] = _i32(np.concatenate([np.arange(n) for n in new]))
    table, _, _, n = _tables(ctx + new, page, rng)
    st["table"] = _i32(table)
    hkv, hd = case["kv_heads"], case["head_dim"]
    if op == "attn":
        st["k"], st["v"] = normal(n, hkv, page, hd), normal(n, hkv, page, hd)
        st["q"] = normal(rows, case["heads"] * hd) * 1.5
        # what lies behind a sequence's last token in its last page was never written
        for i in range(b):
            at = int(ctx[i] + new[i])
            if at % page:
                st["k"][int(table[i, at // page]), :, at % page:] = float("nan")
                st["v"][int(table[i, at // page]), :, at % page:] = float("nan")
        st["out"] = torch.zeros(rows, case["heads"] * hd, device="cuda")
        return st
    st["k"], st["v"] = normal(case["layers"], n, hkv, page, hd), normal(case["layers"], n, hkv, page, hd)
    tokens = rng.integers(0, 128256, rows)
    nxt = rng.integers(0, 128256, rows)
    for i in range(b):  # the deepest node of at most `keep` in its branch is what the model goes along with
        bits = _masks(parents[i])
        depth = [bin(m).count("1") for m in bits]
        at = max((d, -k) for k, d in enumerate(depth) if d <= case["keep"])
        path = [k for k in range(len(bits)) if bits[-at[1]] >> k & 1]
        for p, c in zip(path, path[1:]):
            nxt[start[i] + p] = tokens[start[i] + c]
    st["tokens"] = _i32(tokens)
    score = rng.integers(1 << 31, 1 << 32, rows).astype(np.uint64)
    st["keys"] = torch.from_numpy((score << np.uint64(32) | (np.uint64(0xFFFFFFFF) - nxt.astype(np.uint64))).view(np.int64)).cuda()
    st["path"] = torch.full((b, 64), -1, dtype=torch.int32, device="cuda")
    for k in ("count", "next", "ctx_out"):
        st[k] = torch.zeros(b, dtype=torch.int32, device="cuda")
    return st


# ---- the plain forms --------------------------------------------------------------------------------


def _bits(tree):
    return (tree[:, None] >> torch.arange(64, device="cuda")) & 1


def _plain_attn(st):
    c, page = st["case"], st["page"]
    b, h, hkv, hd = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    grp, length, most = h // hkv, st["longest"], st["most_new"]
    item, local = st["row_item"].long(), st["row_local"].long()
    ctx, new = st["ctx_len"].long(), st["new_len"].long()
    at = torch.arange(length, device="cuda")
    pages = st["table"].long()[:, at // page].clamp(min=0)
    held = (at < (ctx + new)[:, None])[:, :, None, None]
    k = torch.where(held, st["k"][pages, :, at % page], 0.0).permute(0, 2, 3, 1)
    v = torch.where(held, st["v"][pages, :, at % page], 0.0).permute(0, 2, 1, 3)
    q = torch.zeros(b, most, h, hd, device="cuda")
    q[item, local] = st["q"].view(-1, h, hd)
    q = q.view(b, most, hkv, grp, hd).permute(0, 2, 1, 3, 4).reshape(b, hkv, most * grp, hd)
    seen = torch.zeros(b, most, length, dtype=torch.bool, device="cuda")
    behind = at[None] - ctx[item][:, None]
    if st["tree"] is not None:
        drafted = (st["tree"][:, None] >> behind.clamp(0, 63)) & 1 > 0
    else:
        drafted = behind <= local[:, None]
    seen[item, local] = (behind < 0) | (drafted & (behind < new[item][:, None]))
    seen = seen[:, None, :, None, :].expand(b, hkv, most, grp, length).reshape(b, hkv, most * grp, length)
    s = torch.where(seen, (q @ k) / math.sqrt(hd), -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-37)
    o = o.view(b, hkv, most, grp, hd).permute(0, 2, 1, 3, 4).reshape(b, most, h * hd)
    return o[item, local]


def _plain_plan(st):
    page, table = st["page"], st["table"].long()
    ctx, new, mapped = st["ctx_len"].long(), st["new_len"].long(), st["mapped"].long()
    start = torch.zeros(len(new) + 1, dtype=torch.long, device="cuda")
    start[1:] = new.cumsum(0)
    need = torch.maximum((ctx + new + page - 1) // page, mapped)
    fresh = need - mapped
    base = fresh.cumsum(0) - fresh
    logical = torch.arange(table.shape[1], device="cuda")
    rank = base[:, None] + logical - mapped[:, None]
    count = st["free_count"].long()
    page_of = st["free"].long()[(count - 1 - rank).clamp(0, len(st["free"]) - 1)]
    table = torch.where((logical >= mapped[:, None]) & (logical < need[:, None]), page_of, table)
    item = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new, output_size=st["rows"])
    local = torch.arange(st["rows"], device="cuda") - start[item]
    slot_at = ctx[item] + local
    pos = ctx[item] + (_bits(st["tree"]).sum(1) - 1 if st["tree"] is not None else local)
    slot = table[item, slot_at // page] * page + slot_at % page
    return [x.int() for x in (start, item, pos, slot, table, need, count - fresh.sum())]


def _plain_append(st):
    c, page = st["case"], st["page"]
    h, hkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    y = st["y"].view(-1, h + 2 * hkv, hd)
    # the angle is the 32-bit product of position and frequency, as everywhere in this library
    a = (st["positions"].float()[:, None] * st["freq"])[:, None]
    cos, sin = torch.cos(a), torch.sin(a)
    x0, x1 = y[:, :h + hkv, 0::2], y[:, :h + hkv, 1::2]
    r = torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).reshape(-1, h + hkv, hd)
    slot = st["slots"].long()
    st["k"][slot // page, :, slot % page] = r[:, h:]
    st["v"][slot // page, :, slot % page] = y[:, h + hkv:]
    return [r[:, :h].reshape(-1, h * hd), st["k"], st["v"]]


def _plain_accept(st):
    c, page = st["case"], st["page"]
    item, local, new, ctx = (st[k].long() for k in ("row_item", "row_local", "new_len", "ctx_len"))
    most = st["most_new"]
    b, me = c["batch"], torch.arange(most, device="cuda")
    tok, nxt = torch.full((b, most), -1, device="cuda"), torch.full((b, most), -2, device="cuda")
    anc = torch.zeros(b, most, most, dtype=torch.bool, device="cuda")
    tok[item, local] = st["tokens"].long()
    nxt[item, local] = 0xFFFFFFFF - (st["keys"] & 0xFFFFFFFF)
    anc[item, local] = _bits(st["tree"])[:, :most] > 0
    above = anc & (me[None, :] < me[:, None])
    parent = torch.where(above, me, -1).amax(-1)
    fits = tok == torch.gather(nxt, 1, parent.clamp(min=0))
    fits[:, 0] = True
    twin = (parent[:, :, None] == parent[:, None, :]) & (tok[:, :, None] == tok[:, None, :]) & (me[None, :] < me[:, None])
    fits = fits & ~twin.any(-1)
    taken = (~anc | fits[:, None, :]).all(-1) & (me < new[:, None])
    count = taken.sum(-1)
    path = torch.sort(torch.where(taken, me, 64), 1).values
    path = torch.nn.functional.pad(torch.where(path == 64, -1, path), (0, 64 - most), value=-1)
    last = torch.gather(path, 1, count[:, None] - 1)
    follow = torch.gather(nxt, 1, last)[:, 0]
    src = ctx[:, None] + torch.where(path[:, :most] < 0, me, path[:, :most])
    dst = (ctx[:, None] + me).expand(b, most)
    live = (me < new[:, None]).reshape(-1)
    src, dst = torch.where(live, src.reshape(-1), 0), torch.where(live, dst.reshape(-1), 0)
    row = torch.arange(b, device="cuda")[:, None].expand(b, most).reshape(-1)
    table = st["table"].long()
    ps, pd = table[row, src // page], table[row, dst // page]
    for x in (st["k"], st["v"]):
        x[:, pd, :, dst % page] = x[:, ps, :, src % page]
    return [path.int(), count.int(), follow.int(), (ctx + count).int(), st["k"], st["v"]]


# ---- the library --------------------------------------------------------------------------------------


def _library():
    d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "att-1_b200")
    if d not in sys.path:
        sys.path.insert(0, d)
    import att1_b200
    return att1_b200


def _kv(b2, st, k, v):
    c = st["case"]
    table = st.get("table")
    return b2.KVLayout(k, v, table.data_ptr() if table is not None else None, st["page"],
                       table.shape[1] if table is not None else 0, c["kv_heads"], c["head_dim"])


def _arguments(b2, st):
    """The calls' argument structs: a user's program fills them in once and calls again."""
    c, op = st["case"], st["op"]

    def p(name):
        return st[name].data_ptr() if st.get(name) is not None else None

    if op == "attn":
        a = b2.AttnRowsArgs(batch=c["batch"], n_heads=c["heads"], n_kv_heads=c["kv_heads"], head_dim=c["head_dim"],
                            max_rows=st["most_new"], rows=st["rows"], q=p("q"), q_stride=c["heads"] * c["head_dim"],
                            kv=_kv(b2, st, p("k"), p("v")), row_start=p("row_start"), ctx_len=p("ctx_len"),
                            tree=p("tree"), max_ctx=st["longest"], ctx=p("out"), ctx_stride=c["heads"] * c["head_dim"],
                            err=p("err"), pdl=1)
        need = b2.lib().b2_attn_rows_scratch_bytes(a)
        st["scratch"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        a.scratch, a.scratch_bytes = p("scratch"), need
        return a
    if op == "plan":
        return b2.KvPlanArgs(batch=c["batch"], max_rows=st["rows"], page_tokens=st["page"],
                             pages_per_seq=st["table"].shape[1], pool_pages=st["pool_pages"], ctx_len=p("ctx_len"),
                             new_len=p("new_len"), tree=p("tree"), mapped=p("mapped"), free_pages=p("free"),
                             free_count=p("free_count"), page_table=p("table"), mapped_out=p("mapped_out"),
                             free_out=p("free_out"), row_start=p("row_start"), row_item=p("row_item"),
                             row_pos=p("row_pos"), row_slot=p("row_slot"), err=p("err"), pdl=1)
    if op == "append":
        return b2.RowsAppendArgs(m=c["rows"], y=p("y"), y_stride=st["y"].shape[1], q_rows=c["heads"] * c["head_dim"],
                                 q=p("q"), q_stride=st["q"].shape[1], rope_freq=p("freq"), positions=p("positions"),
                                 slots=p("slots"), kv=_kv(b2, st, p("k"), p("v")), pool_pages=st["k"].shape[0],
                                 err=p("err"), pdl=1)
    a = b2.TreeAcceptArgs(batch=c["batch"], max_rows=st["most_new"], rows=st["rows"], row_start=p("row_start"),
                          tokens=p("tokens"), tree=p("tree"), argmax=p("keys"), ctx_len=p("ctx_len"), path=p("path"),
                          count=p("count"), next=p("next"), ctx_out=p("ctx_out"), err=p("err"), pdl=1)
    layer = st["k"][0].numel() * 4
    kvs = (b2.KVLayout * c["layers"])(*[_kv(b2, st, p("k") + i * layer, p("v") + i * layer) for i in range(c["layers"])])
    m = b2.KvCompactArgs(n_layers=c["layers"], layers=kvs, batch=c["batch"], ctx_len=p("ctx_len"), path=p("path"),
                         count=p("count"), err=p("err"), pdl=1)
    return a, m


def _own(st):
    b2 = _library()
    if "args" not in st:
        st["args"] = _arguments(b2, st)
    a, stream, lib = st["args"], torch.cuda.current_stream().cuda_stream, b2.lib()
    if st["op"] == "attn":
        b2.check("b2_attn_rows", lib.b2_attn_rows(a, stream))
        return st["out"]
    if st["op"] == "plan":
        b2.check("b2_kv_plan", lib.b2_kv_plan(a, stream))
        return [st[k] for k in ("row_start", "row_item", "row_pos", "row_slot", "table", "mapped_out", "free_out")]
    if st["op"] == "append":
        b2.check("b2_rows_append", lib.b2_rows_append(a, stream))
        return [st["q"], st["k"], st["v"]]
    b2.check("b2_tree_accept", lib.b2_tree_accept(a[0], stream))
    b2.check("b2_kv_compact", lib.b2_kv_compact(a[1], stream))
    return [st[k] for k in ("path", "count", "next", "ctx_out", "k", "v")]


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "plan": _plain_plan, "append": _plain_append, "accept": _plain_accept}[state["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "append":
        h, hkv, hd, rows = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
        return {"bytes": 8 * rows * (h + 2 * hkv) * hd + 8 * rows, "flops": 3 * rows * (h + hkv) * hd}
    ctx, new = _lengths(case)
    b, rows = len(new), int(new.sum())
    if op == "attn":
        h, hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        # a tree's rows see the cache and a branch of about the logarithm of the tree's size
        keys = int((new * ctx).sum()) + (rows * math.log2(rows / b + 1) if case["tree"] else float((new * (new + 1) / 2).sum()))
        return {"bytes": 8 * hkv * hd * int((ctx + new).sum()) + 8 * rows * h * hd + 8 * rows * case["tree"], "flops": 4 * h * hd * keys}
    if op == "plan":
        page = case["page"]
        fresh = int((-(-(ctx + new) // page) - -(-ctx // page)).sum())
        return {"bytes": rows * (12 + 8 * case["tree"]) + 20 * b + 8 * fresh + 4 * int((-(-ctx // page) - ctx // page).sum()), "flops": rows * 8}
    moved = max(case["keep"] - 1, 0)
    return {"bytes": rows * 20 + b * 280 + 16 * b * moved * case["layers"] * case["kv_heads"] * case["head_dim"], "flops": rows * 8}


# ---- the definitions in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attn":
        h, hkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        grp = h // hkv
        out = torch.empty(st["rows"], h, hd, dtype=torch.float64, device="cuda")
        first = st["row_start"].tolist()
        ctx = st["ctx_len"].tolist()
        table = st["table"].cpu()
        for i in range(case["batch"]):
            n, held = first[i + 1] - first[i], ctx[i] + first[i + 1] - first[i]
            pages = table[i, :-(-held // page)].long().cuda()
            q = st["q"][first[i]:first[i + 1]].double().view(n, h, hd)
            allowed = torch.ones(n, held, dtype=torch.bool, device="cuda")
            if st["tree"] is None:
                allowed[:, ctx[i]:] = torch.ones(n, n, device="cuda").tril() > 0
            else:
                allowed[:, ctx[i]:] = torch.tensor([[m >> j & 1 for j in range(n)] for m in st["tree"][first[i]:first[i + 1]].tolist()], device="cuda") > 0
            for kv in range(hkv):
                k = st["k"][pages, kv].reshape(-1, hd)[:held].double()
                v = st["v"][pages, kv].reshape(-1, hd)[:held].double()
                for j in range(kv * grp, (kv + 1) * grp):
                    s = (q[:, j] @ k.T * hd ** -0.5).masked_fill(~allowed, -math.inf)
                    out[first[i]:first[i + 1], j] = torch.softmax(s, -1) @ v
        return out.view(st["rows"], h * hd)
    if case["op"] == "append":
        h, hkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        y = st["y"].double().view(-1, h + 2 * hkv, hd)
        angle = (st["positions"].float()[:, None] * st["freq"][None]).double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        z = torch.view_as_real(torch.view_as_complex(y[:, :h + hkv].reshape(-1, h + hkv, hd // 2, 2).contiguous()) * turn)
        z = z.reshape(-1, h + hkv, hd)
        flat = [x.double().transpose(1, 2).reshape(-1, hkv, hd) for x in (st["k"], st["v"])]
        flat[0][st["slots"].long()], flat[1][st["slots"].long()] = z[:, h:], y[:, h + hkv:]
        k, v = (x.view(-1, page, hkv, hd).transpose(1, 2) for x in flat)
        return [z[:, :h].reshape(-1, h * hd), k, v]
    return None
