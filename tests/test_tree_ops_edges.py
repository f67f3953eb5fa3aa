"""Edges of the operators of several new rows per sequence: masks and paths that
no tree has, batch sizes at the default shared-memory limit, rows in use counted
by the kernel before, and the attention kernels' values that are not finite, of
very different sizes, or far from 1.

Tolerances of the attention: with A the largest scale * sum |q_i k_i| of a row
and a place, a score is off by at most A 2^-21 (2^-22 for the operands, as much for the
f32 sums) and, where an operand is far below its neighbours, by
scale * 2^-25 * (sum |q_i| + sum |k_i|); a weight by twice that relative to its softmax, and
an output by as much of sum_j p_j |v_j|. Of that sum the products and sums take another
2^-19: 2^-21 each for the weights' 21 bits, the product of the two low parts
that is left out and the f32 sums, 2^-22 each for V's 22 bits and the exponential. An
element of V far below its neighbours keeps 2^-25 (of 1 where the largest of
them lies between 2^-4 and 2^12), the weights' low parts less than that together.
"""
import subprocess
import sys

import numpy as np
import pytest

from test_tree_ops import (ATTN_TOL, ERR_NONFINITE, ERR_POSITION, ERR_TREE, Scene, accept_run, compact_run, dev, p, plan_case,
                           plan_check, plan_run)

pytestmark = pytest.mark.gpu

# shapes that each of the attention's three kernels takes: up to 16 rows of a KV head, blocks of 128, four of them and more
FEW, ROWS, LAID = [(4, 2, 64, 7), (2, 1, 128, 8), (3, 1, 48, 5)], [(4, 2, 64, 20), (8, 2, 128, 24), (4, 1, 48, 64)], [(8, 1, 128, 64), (16, 2, 64, 64)]


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.init()
    return torch


def exact(s, hide=()):
    """Outputs in float64 without the places of `hide`; sum_j p_j |v_j|; the bound of a weight's relative error; the least gap
    of a row's two best scores."""
    out = np.zeros((s.rows, s.h, s.hd))
    size, rel, gap = np.zeros_like(out), 0.0, np.inf
    g, scale = s.h // s.hkv, 1 / np.sqrt(s.hd)
    for b in range(s.batch):
        t = int(s.ctx[b] + s.new[b])
        pg, off = s.table[b, np.arange(t) // s.page], np.arange(t) % s.page
        K, V = s.k[pg, :, off].astype(np.float64), s.v[pg, :, off].astype(np.float64)
        for i in range(int(s.new[b])):
            at = [j for j in s.sees(b, i) if j not in hide]
            q = s.q[s.start[b] + i, :s.h * s.hd].astype(np.float64).reshape(s.hkv, g, s.hd)
            x = np.einsum("hgd,thd->hgt", q, K[at]) * scale
            top = np.sort(x, -1)
            gap = min(gap, (top[..., -1] - top[..., -2]).min())
            w = np.exp(x - x.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            r = s.start[b] + i
            out[r] = np.einsum("hgt,thd->hgd", w, V[at]).reshape(s.h, s.hd)
            size[r] = np.einsum("hgt,thd->hgd", w, np.abs(V[at])).reshape(s.h, s.hd)
            a = np.einsum("hgd,thd->hgt", np.abs(q), np.abs(K[at])).max() * scale
            rel = max(rel, 2 * (a * 2.0 ** -21 + scale * 2.0 ** -25 * (np.abs(q).sum(-1).max() + np.abs(K[at]).sum(-1).max())))
    return out, size, rel, gap


# ---- attention --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("victim", [1, 2, 4, 6])
@pytest.mark.parametrize("h,hkv,hd,new", FEW[:2])
def test_attn_few_rows_masked_places_may_hold_anything(b2, torch, h, hkv, hd, new, victim, which, bad):
    """Places 38 to 43: both halves of a unit of 16, and neighbouring columns of a lane."""
    s = Scene(torch, h, hkv, hd, 16, [37], [new], seed=13)
    ref = s.reference()
    pg, off = s.place(0, 37 + victim)
    getattr(s, which)[pg, hkv - 1, off, 5] = bad
    got, err = s.run(b2)
    first = (hkv - 1) * (h // hkv)   # heads of the KV head that holds it
    seen = [bool(s.masks[i] >> victim & 1) for i in range(new)]
    assert any(seen) and not all(seen) and err == ERR_NONFINITE
    for i in range(new):
        assert np.abs(got[i, :first] - ref[i, :first]).max(initial=0) <= ATTN_TOL * 5
        if seen[i]:
            assert np.isnan(got[i, first:]).all()
        else:
            assert np.abs(got[i, first:] - ref[i, first:]).max() <= ATTN_TOL * 5


@pytest.mark.parametrize("at", [0, 3, 20, 31, 36])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("h,hkv,hd,new", FEW)
def test_attn_few_rows_nonfinite_cached_place(b2, torch, h, hkv, hd, new, which, at):
    """A cached place is seen by every row."""
    s = Scene(torch, h, hkv, hd, 16, [37], [new], seed=14)
    ref = s.reference()
    pg, off = s.place(0, at)
    getattr(s, which)[pg, 0, off, hd - 1] = np.nan
    got, err = s.run(b2)
    assert err == ERR_NONFINITE and np.isnan(got[:, :h // hkv]).all()
    assert np.abs(got[:, h // hkv:] - ref[:, h // hkv:]).max(initial=0) <= ATTN_TOL * 5


@pytest.mark.parametrize("big", [3e3, 1e5, 1e10, 1e30, 3e38])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("victim", [1, 2, 4, 6])
@pytest.mark.parametrize("h,hkv,hd,new", FEW[:2])
def test_attn_few_rows_hidden_place_takes_no_precision(b2, torch, h, hkv, hd, new, victim, which, big):
    s = Scene(torch, h, hkv, hd, 16, [37], [new], seed=13)
    ref = s.reference()
    pg, off = s.place(0, 37 + victim)
    getattr(s, which)[pg, :, off] = big * np.sign(getattr(s, which)[pg, :, off])
    got, _ = s.run(b2)
    hidden = [i for i in range(new) if not s.masks[i] >> victim & 1]
    assert hidden
    assert np.abs(got[hidden] - ref[hidden]).max() <= ATTN_TOL * 5


@pytest.mark.parametrize("at", [5, 12, 20, 31, 36])
@pytest.mark.parametrize("h,hkv,hd,new", FEW)
def test_attn_few_rows_place_of_no_weight_takes_no_precision(b2, torch, h, hkv, hd, new, at):
    """A cached place whose K is 2^14 times the others' in one direction and whose V is 2^40."""
    s = Scene(torch, h, hkv, hd, 16, [37], [new], seed=16)
    pg, off = s.place(0, at)
    s.k[pg, :, off] = 0
    s.k[pg, :, off, 3] = 2.0 ** 14
    s.v[pg, :, off] = 2.0 ** 40
    q = s.q[:s.rows, :h * hd].reshape(s.rows, h, hd)
    q[:, :, 3] = np.where(q[:, :, 3] > 0, 1, -1)  # scores of +-2^14 / sqrt(hd)
    got, err = s.run(b2)
    drawn = q[:, :, 3] > 0
    assert err == 0 and drawn.any() and not drawn.all()
    assert (np.abs(got[drawn] - 2.0 ** 40) <= ATTN_TOL * 2.0 ** 40).all()
    others = exact(s, hide=(at,))[0]
    assert np.abs(got[~drawn] - others[~drawn]).max() <= ATTN_TOL * 5


@pytest.mark.parametrize("growing", [True, False, None])
@pytest.mark.parametrize("h,hkv,hd,new", FEW + ROWS + LAID)
def test_attn_saturated_softmax(b2, torch, h, hkv, hd, new, growing):
    """Scores past +-60, every place's K times a power of two of its own from 2^-6 to 2^3, growing along the places (the maximum
    rises from tile to tile and the sums are rescaled), falling, or in no order."""
    s = Scene(torch, h, hkv, hd, 16, [300], [new], seed=21)
    t = 300 + new
    size = np.floor(np.arange(t) * 9.99 / t).astype(int) - 6
    if growing is None:
        size = np.random.default_rng(5).permutation(size)
    elif not growing:
        size = size[::-1]
    pg, off = s.table[0, np.arange(t) // 16], np.arange(t) % 16
    s.k[pg, :, off] *= np.ldexp(np.float32(1), size)[:, None, None]
    s.q *= np.float32(6)
    ref, mean, rel, _ = exact(s)
    top = np.einsum("hgd,thd->hgt", s.q[0, :h * hd].reshape(hkv, h // hkv, hd), s.k[pg[:300], :, off[:300]]) / np.sqrt(hd)
    assert np.abs(top).max() > 60
    got, err = s.run(b2)
    assert err == 0
    assert (np.abs(got - ref) <= (rel + 2.0 ** -19) * mean.max(-1, keepdims=True) + 2.0 ** -24).all()


@pytest.mark.parametrize("h,hkv,hd,new", FEW + ROWS + LAID)
def test_attn_small_channels(b2, torch, h, hkv, hd, new):
    """Dimension d of V times 2^-(d mod 16): every dimension keeps its own bound, 2^-25 of 1 at the finest."""
    s = Scene(torch, h, hkv, hd, 16, [150], [new], seed=22)
    s.v *= np.ldexp(np.float32(1), -(np.arange(hd) % 16))
    ref, mean, rel, _ = exact(s)
    got, err = s.run(b2)
    assert err == 0
    assert (np.abs(got - ref) <= (rel + 2.0 ** -19) * mean + 2.0 ** -24).all()


@pytest.mark.parametrize("size_q,size_k", [(10, 12), (12, 12), (11, 14), (13, 14), (16, 15), (30, 30), (60, -25), (-25, 60)])
@pytest.mark.parametrize("h,hkv,hd,new", FEW + ROWS + LAID)
def test_attn_scores_of_any_size(b2, torch, h, hkv, hd, new, size_q, size_k):
    """Scores of 2^23 to 2^61: where one place is ahead by more than they can be off, its V comes out."""
    s = Scene(torch, h, hkv, hd, 16, [61], [new], seed=24)
    s.q *= np.float32(2.0 ** size_q)
    s.k *= np.float32(2.0 ** size_k)
    ref, _, _, gap = exact(s)
    assert gap > 0
    t = 61 + new
    pg, off = s.table[0, np.arange(t) // 16], np.arange(t) % 16
    got, err = s.run(b2)
    assert err == 0
    clear = 0
    for i in range(new):
        at = s.sees(0, i)
        for hh in range(h):
            q, K = s.q[i, hh * hd:(hh + 1) * hd].astype(np.float64), s.k[pg[at], hh // (h // hkv), off[at]].astype(np.float64)
            x, a = K @ q / np.sqrt(hd), (np.abs(K) @ np.abs(q)).max() / np.sqrt(hd)
            if np.diff(np.sort(x)[-2:])[0] > 2 * a * 2.0 ** -21 + 32:   # the second's weight is below 2^-46
                clear += 1
                assert np.abs(got[i, hh] - ref[i, hh]).max() <= 2.0 ** -19 * np.nanmax(np.abs(s.v))
    assert clear > 0.95 * new * h


@pytest.mark.parametrize("h,hkv,hd,new", FEW + ROWS + LAID)
def test_attn_scores_in_range_of_operands_far_from_one(b2, torch, h, hkv, hd, new):
    """q of 2^126 and K of 2^-90, some places 2^-98 and one hidden from some rows 2^13: scores of 2^36, one weight takes all."""
    s = Scene(torch, h, hkv, hd, 16, [61], [new], seed=23)
    t = 61 + new
    victim = 3
    s.q = (np.sign(s.q) * np.float32(2.0 ** 126) * (1 + np.abs(s.q) / 16)).astype(np.float32)
    s.k *= np.float32(2.0 ** -90)
    for j in range(t):
        if j % 24 < 8:
            pg, off = s.place(0, j)
            s.k[pg, :, off] *= np.float32(2.0 ** -8)
    pg, off = s.place(0, 61 + victim)
    s.k[pg, :, off] = np.sign(s.k[pg, :, off]) * 2.0 ** 13
    rows = [i for i in range(new) if not s.masks[i] >> victim & 1]
    assert rows and np.isfinite(s.q).all()
    ref, _, _, gap = exact(s, hide=(61 + victim,))
    assert gap > 2.0 ** 20   # against an error of about 2^37 2^-21
    got, _ = s.run(b2)
    assert np.abs(got[rows] - ref[rows]).max() <= 2.0 ** -19 * np.nanmax(np.abs(s.v))


@pytest.mark.parametrize("h,hkv,hd,new", [(8, 2, 128, 24), (10, 2, 80, 20), (8, 2, 64, 24)])
def test_attn_pages_far_apart(b2, torch, h, hkv, hd, new):
    """Every page 64 MB from the next, so the copies of K and V come in at times of their own, in an order other than they were
    asked for; the same bits each time."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough device memory free")
    page = 16
    s = Scene(torch, h, hkv, hd, page, [1500, 700], [new, new], seed=25)
    a = s.args(b2)
    stride = (64 << 20) // (hkv * page * hd * 4)
    used = np.unique(s.table[s.table >= 0])
    k, v = (torch.empty(stride * (s.pool_pages + 1), hkv, page, hd, device="cuda") for _ in range(2))
    at = dev(torch, used, np.int64)
    k[at * stride], v[at * stride] = s.d["k"][at], s.d["v"][at]
    far = dev(torch, np.where(s.table >= 0, s.table * stride, s.table), np.int32)
    a.kv.k_pool, a.kv.v_pool, a.kv.page_table, a.pool_pages = p(k), p(v), p(far), k.shape[0]
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    ref, first = s.reference(), None
    for _ in range(12):
        flush.zero_()
        s.d["out"].zero_()
        assert b2.lib().b2_attn_rows(a, None) == 0
        torch.cuda.synchronize()
        got = s.d["out"].cpu().numpy()[:s.rows, :h * hd].reshape(s.rows, h, hd)
        assert int(s.d["err"].item()) == 0 and np.abs(got - ref).max() <= ATTN_TOL * 5
        assert first is None or (got == first).all()
        first = got


@pytest.mark.parametrize("h,hkv,hd,new", [(8, 1, 128, [130, 64]), (8, 2, 64, [200, 40]), (8, 2, 128, [20, 31]), (4, 2, 64, [6, 8])])
def test_attn_layers_share_q_and_scratch(b2, torch, h, hkv, hd, new):
    """Append and attention of eight layers through one q buffer and one scratch, each kernel launched while the one before still
    runs, captured and replayed: the bits of each layer by itself."""
    L, layers, page, batch = b2.lib(), 8, 16, len(new)
    rng = np.random.default_rng(hd + h)
    ctx, rows = [150, 37], sum(new)
    start = np.concatenate([[0], np.cumsum(new)])
    pps = max(-(-(c + n) // page) for c, n in zip(ctx, new))
    pool = batch * pps
    tab = rng.permutation(pool).reshape(batch, pps)
    slot = [int(tab[b, (ctx[b] + i) // page]) * page + (ctx[b] + i) % page for b in range(batch) for i in range(new[b])]
    d = dict(start=dev(torch, start, np.int32), ctx=dev(torch, ctx, np.int32), table=dev(torch, tab, np.int32), slot=dev(torch, slot, np.int32))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    y = torch.randn(layers, rows, (h + 2 * hkv) * hd, generator=g, device="cuda")
    k, v = (torch.randn(layers, pool, hkv, page, hd, generator=g, device="cuda") for _ in range(2))
    q, o = torch.zeros(rows, h * hd, device="cuda"), torch.zeros(layers, rows, h * hd, device="cuda")
    scratch = None

    def layer(i, stream, pdl):
        nonlocal scratch
        kv = b2.KVLayout(p(k[i]), p(v[i]), p(d["table"]), page, pps, hkv, hd)
        b2.check("append", L.b2_rows_append(b2.RowsAppendArgs(m=rows, y=p(y[i]), y_stride=y.shape[2], q_rows=h * hd, q=p(q), q_stride=h * hd,
                                                              slots=p(d["slot"]), kv=kv, pool_pages=pool, err=p(err), pdl=pdl), stream))
        a = b2.AttnRowsArgs(batch=batch, n_heads=h, n_kv_heads=hkv, head_dim=hd, max_rows=max(new), rows=rows, q=p(q), q_stride=h * hd, kv=kv,
                            pool_pages=pool, row_start=p(d["start"]), ctx_len=p(d["ctx"]), max_ctx=pps * page, ctx=p(o[i]),
                            ctx_stride=h * hd, err=p(err), pdl=pdl)
        need = L.b2_attn_rows_scratch_bytes(a)
        if scratch is None:
            scratch = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
        a.scratch, a.scratch_bytes = p(scratch), need
        b2.check("attn", L.b2_attn_rows(a, stream))

    for i in range(layers):
        layer(i, None, 0)
        torch.cuda.synchronize()
    want = o.clone()
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        for i in range(layers):
            layer(i, torch.cuda.current_stream().cuda_stream, 1)
    for _ in range(20):
        o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0 and (o == want).all()


# ---- b2_kv_plan, b2_rows_append -----------------------------------------------------------------------------


BATCHES = """
import sys
sys.path[:0] = {path!r}
import numpy as np, torch, att1_b200 as b2
from test_tree_ops import plan_case, plan_check
torch.cuda.init()
for batch in (3055, 3056, 3070):
    rng = np.random.default_rng(batch)
    plan_check(b2, torch, plan_case(torch, rng.integers(0, 50, batch), rng.integers(0, 8, batch), 16, batch % 2 == 0, seed=batch))
"""


def test_plan_batches_at_the_shared_memory_limit():
    """In a process of its own: a larger batch raises the kernel's limit for those after it."""
    r = subprocess.run([sys.executable, "-c", BATCHES.format(path=sys.path)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_plan_mask_without_a_row(b2, torch):
    """An empty mask is no tree's: reported, and the row's position is not before the new rows."""
    for ctx in ([0, 20], [7, 0]):
        c = plan_case(torch, ctx, [3, 4], 16, True)
        want = plan_run(b2, torch, c)
        c["masks"][1] = c["masks"][5] = 0
        got = plan_run(b2, torch, c)
        assert want["err"][0] == 0 and got["err"][0] == ERR_TREE
        pos = want["pos"].copy()
        pos[1], pos[5] = ctx[0], ctx[1]
        assert (got["pos"] == pos).all()
        for k in ("item", "slot", "start", "table", "mo", "fo"):
            assert (got[k] == want[k]).all()


def test_append_takes_as_many_rows_as_the_plan_before_it(b2, torch):
    """Plan and append captured together, the second launched while the first runs: the rows in use are those of this replay."""
    h, hkv, hd, page, batch, cap = 4, 2, 64, 16, 3, 24
    pool = 12
    L = b2.lib()
    rng = np.random.default_rng(3)
    y = dev(torch, rng.normal(0, 1, (cap, (h + 2 * hkv) * hd)), np.float32)
    table, free = dev(torch, np.full((batch, 4), -1), np.int32), dev(torch, rng.permutation(pool), np.int32)
    i32 = {k: torch.zeros(n, dtype=torch.int32, device="cuda") for k, n in dict(
        ctx=batch, new=batch, mapped=batch, mo=batch, fo=1, start=batch + 1, item=cap, pos=cap, slot=cap, err=1).items()}
    count = dev(torch, [pool], np.int32)
    q = torch.zeros(cap, h * hd, device="cuda")
    k, v = (torch.zeros(pool, hkv, page, hd, device="cuda") for _ in range(2))
    plan = b2.KvPlanArgs(batch=batch, max_rows=cap, page_tokens=page, pages_per_seq=4, pool_pages=pool, ctx_len=p(i32["ctx"]),
                         new_len=p(i32["new"]), mapped=p(i32["mapped"]), free_pages=p(free), free_count=p(count), page_table=p(table),
                         mapped_out=p(i32["mo"]), free_out=p(i32["fo"]), row_start=p(i32["start"]), row_item=p(i32["item"]),
                         row_pos=p(i32["pos"]), row_slot=p(i32["slot"]), err=p(i32["err"]), pdl=1)
    app = b2.RowsAppendArgs(m=cap, y=p(y), y_stride=y.shape[1], q_rows=h * hd, q=p(q), q_stride=h * hd, slots=p(i32["slot"]),
                            n_rows=i32["start"].data_ptr() + 4 * batch, kv=b2.KVLayout(p(k), p(v), None, page, 0, hkv, hd),
                            pool_pages=pool, err=p(i32["err"]), pdl=1)

    def step(stream):
        b2.check("plan", L.b2_kv_plan(plan, stream))
        b2.check("append", L.b2_rows_append(app, stream))

    st = torch.cuda.Stream()
    step(st.cuda_stream)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        step(torch.cuda.current_stream().cuda_stream)
    for new in ([1, 0, 2], [8, 8, 8], [0, 0, 0], [5, 1, 0], [2, 20, 2]):
        i32["new"].copy_(dev(torch, new, np.int32))
        q.fill_(7.25)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        n = sum(new)
        assert int(i32["err"].item()) == 0 and int(i32["start"][batch].item()) == n
        assert (q[:n] == y[:n, :h * hd]).all() and (q[n:] == 7.25).all()


# ---- b2_tree_accept, b2_kv_compact ----------------------------------------------------------------------------


@pytest.mark.parametrize("masks,count,follow", [
    ([1, 3, 7, 13], 1, 4),          # row 3 below row 2 without row 2's other ancestor; the root's token is nobody's
    ([1, 3, 7, 15], 1, 4),          # the same tokens in a proper chain
    ([1, 3, 5, 11, 31], 1, 4),      # row 4 has two branches' rows
])
def test_accept_masks_that_are_not_their_parents(b2, torch, masks, count, follow):
    tokens, nxt = [9, 5, 6, 7, 8][:len(masks)], [4, 6, 7, 8, 3][:len(masks)]
    r = accept_run(b2, torch, [0, len(masks)], tokens, masks, nxt, [11])
    proper = all(m >> i == 1 and (i == 0 or m ^ 1 << i == masks[(m ^ 1 << i).bit_length() - 1]) for i, m in enumerate(masks))
    assert r["err"][0] == (0 if proper else ERR_TREE)
    assert r["count"][0] == count and r["next"][0] == follow and r["out"][0] == 11 + count
    assert list(r["path"][0][:count + 1]) == [0, -1]


def test_accept_stops_before_a_mask_that_is_not_its_parents(b2, torch):
    """Rows that fit by their tokens: the branch ends before the row whose mask omits an ancestor, here and past row 32; other
    items are as they were."""
    r = accept_run(b2, torch, [0, 4, 6], [0, 1, 2, 3, 0, 1], [1, 3, 7, 13, 1, 3], [1, 2, 3, 4, 1, 2], [0, 5])
    assert r["err"][0] == ERR_TREE
    assert list(r["count"]) == [3, 2] and list(r["next"]) == [3, 2] and list(r["out"]) == [3, 7]
    masks = [(2 << i) - 1 for i in range(64)]
    masks[40] &= ~(1 << 7)
    r = accept_run(b2, torch, [0, 64], list(range(64)), masks, list(range(1, 65)), [0])
    # row 41's mask is no longer its parent's and its own bit either
    assert r["err"][0] == ERR_TREE and r["count"][0] == 40 and r["next"][0] == 40


@pytest.mark.parametrize("path,moved", [([0, 5, 3], [0, 5]), ([0, 5, 5], [0, 5]), ([4, 3, 9], [4, None, 9]), ([0, -1, 7], [0, None, 7])])
def test_compact_paths_that_do_not_ascend(b2, torch, path, moved):
    got, want, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [path], mutate=None)
    assert err == ERR_POSITION
    # the same call without the refused entries: each is left out by naming its own place
    kept = [i if j is None else j for i, j in enumerate(moved)]
    same, want, _ = compact_run(b2, torch, 2, 2, 64, 16, [10], [kept])
    assert (same == want).all() and (got == want).all()


def test_compact_moves_what_lies_32_entries_behind_a_refused_one(b2, torch):
    """A thread looks up entries i and i + 32: each is refused or moved for itself."""
    path = [2 * i for i in range(8)] + list(range(20, 52))   # entry i of 8 and more is 12 + i
    path[5] = path[4]
    got, _, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [path])
    assert err == ERR_POSITION
    path[5] = 5   # its own place: nothing to move
    same, want, _ = compact_run(b2, torch, 2, 2, 64, 16, [10], [path])
    assert (got == want).all()


def test_compact_pools_past_32_bits_of_places(b2, torch):
    """K and V in one buffer of more than 2^32 places, V's pages one behind K's: no place belongs to both."""
    page, n = 1 << 16, (1 << 16) + 4
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough device memory free")
    pool = torch.empty(n, page, 4, device="cuda")
    pages = [n - 3, 2]
    table = dev(torch, [pages], np.int32)
    rows = torch.arange(80, dtype=torch.float32, device="cuda").reshape(2, 10, 4) + 1
    for x in (0, 1):   # places page - 3 .. page + 6 of the sequence
        pool[pages[0] + x, page - 3:], pool[pages[1] + x, :7] = rows[x, :3], rows[x, 3:]
    path = torch.full((1, 64), -1, dtype=torch.int32, device="cuda")
    path[0, :4] = dev(torch, [0, 2, 5, 9], np.int32)
    kv = (b2.KVLayout * 1)(b2.KVLayout(p(pool), pool[1].data_ptr(), p(table), page, 2, 1, 4))
    d = dict(ctx=dev(torch, [page - 3], np.int32), count=dev(torch, [4], np.int32), err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert b2.lib().b2_kv_compact(b2.KvCompactArgs(n_layers=1, layers=kv, pool_pages=n - 1, batch=1, ctx_len=p(d["ctx"]), path=p(path),
                                                   count=p(d["count"]), err=p(d["err"])), None) == 0
    torch.cuda.synchronize()
    assert int(d["err"].item()) == 0
    for x in (0, 1):
        assert (pool[pages[0] + x, page - 3:] == rows[x, [0, 2, 5]]).all()
        assert (pool[pages[1] + x, 0] == rows[x, 9]).all() and (pool[pages[1] + x, 1:7] == rows[x, 4:]).all()
