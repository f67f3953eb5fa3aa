"""Several new rows per sequence over the paged cache (drafted trees, prompt
chunks): b2_kv_plan, b2_rows_append, b2_attn_rows, b2_tree_accept and
b2_kv_compact through the C ABI against plain numpy / float64 forms.

Tolerances. Integers and moved K/V are exact. Append: one f32 rotation, three
roundings of 2^-24 relative to the pair's length plus sincosf's 2 ulp: 2^-21 of
the largest |y|. Attention: the kernel keeps products to 2^-22 of |q||k| and sums in f32, so a
score is off by at most d = scale * sum |q_i k_i| * (2^-22 + 2^-22) (products,
and a sum of at most 128 terms whose error grows like its square root, 11 half
ulps), a weight by 2 d relative to its softmax, an output by 2 d max|v| plus
2^-20 max|v| for the weighted sum: ATTN_TOL takes sum |q_i k_i| * scale <= 32,
which every input here satisfies (checked).
"""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ATTN_TOL = 2 * 32 * 2.0 ** -21 + 2.0 ** -20   # of max|v|: 3.1e-5
ERR_POSITION, ERR_NONFINITE, ERR_CAPACITY, ERR_TREE = 0x4, 0x2, 0x20, 0x40


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.init()
    return torch


def dev(torch, a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def p(t):
    return None if t is None else t.data_ptr()


def make_tree(n, rng):
    parents = [-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, n)]
    masks = []
    for i, par in enumerate(parents):
        masks.append((masks[par] if par >= 0 else 0) | (1 << i))
    return parents[:n], masks[:n]


class Scene:
    """Sequences over shuffled pages; every place no row may read holds NaN."""

    def __init__(self, torch, h, hkv, hd, page, ctx, new, tree=True, seed=0, slack=1, q_pad=0, spare_rows=3):
        rng = np.random.default_rng(seed)
        self.torch, self.h, self.hkv, self.hd, self.page = torch, h, hkv, hd, page
        self.ctx, self.new = np.array(ctx), np.array(new)
        self.batch = len(ctx)
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.rows = int(self.start[-1])
        total = self.ctx + self.new
        self.pps = int(max(1, (-(-total // page)).max())) + slack
        n = int((-(-total // page)).sum()) + 3
        order = rng.permutation(n)
        self.pool_pages = n
        self.table = np.full((self.batch, self.pps), -7, np.int32)
        at = 0
        for b, t in enumerate(total):
            u = -(-t // page)
            self.table[b, :u] = order[at:at + u]
            at += u
        self.k = np.full((n, hkv, page, hd), np.nan, np.float32)
        self.v = np.full((n, hkv, page, hd), np.nan, np.float32)
        for b, t in enumerate(total):
            for j in range(t):
                self.k[self.table[b, j // page], :, j % page] = rng.normal(0, 1, (hkv, hd))
                self.v[self.table[b, j // page], :, j % page] = rng.normal(0, 1, (hkv, hd))
        self.q_stride = h * hd + q_pad
        self.q = rng.normal(0, 1, (max(self.rows, 1) + spare_rows, self.q_stride)).astype(np.float32)
        self.masks = [m for t in self.new for m in make_tree(int(t), rng)[1]] if tree else None

    def place(self, b, j):
        return self.table[b, j // self.page], j % self.page

    def sees(self, b, i):
        c = int(self.ctx[b])
        m = self.masks[self.start[b] + i] if self.masks is not None else (1 << (i + 1)) - 1
        return list(range(c)) + [c + j for j in range(int(self.new[b])) if m >> j & 1]

    def reference(self):
        out = np.zeros((self.rows, self.h, self.hd))
        g = self.h // self.hkv
        for b in range(self.batch):
            t = int(self.ctx[b] + self.new[b])
            pg, off = self.table[b, np.arange(t) // self.page], np.arange(t) % self.page
            K, V = self.k[pg, :, off].astype(np.float64), self.v[pg, :, off].astype(np.float64)  # [t, hkv, hd]
            for i in range(int(self.new[b])):
                at = self.sees(b, i)
                if not at:
                    continue
                q = self.q[self.start[b] + i, :self.h * self.hd].astype(np.float64).reshape(self.hkv, g, self.hd)
                prod = np.einsum("hgd,thd->hgtd", q, K[at]) if len(at) < 400 else None
                if prod is not None:
                    assert (np.abs(prod).sum(-1).max(initial=0) / np.sqrt(self.hd)) <= 32
                s = np.einsum("hgd,thd->hgt", q, K[at]) / np.sqrt(self.hd)
                w = np.exp(s - s.max(-1, keepdims=True))
                out[self.start[b] + i] = (np.einsum("hgt,thd->hgd", w, V[at]) / w.sum(-1)[..., None]).reshape(self.h, self.hd)
        return out

    def args(self, b2, **over):
        torch = self.torch
        self.d = dict(q=dev(torch, self.q), k=dev(torch, self.k), v=dev(torch, self.v), table=dev(torch, self.table),
                      start=dev(torch, self.start), ctx=dev(torch, self.ctx, np.int32),
                      err=torch.zeros(1, dtype=torch.int32, device="cuda"),
                      out=torch.full((self.q.shape[0], self.h * self.hd + 4), 7.25, device="cuda"))
        if self.masks is not None:
            self.d["tree"] = dev(torch, np.array(list(self.masks) + [0], np.uint64).view(np.int64))
        d = self.d
        a = b2.AttnRowsArgs(batch=self.batch, n_heads=self.h, n_kv_heads=self.hkv, head_dim=self.hd,
                            max_rows=int(max(1, self.new.max())), rows=max(1, self.rows), q=p(d["q"]), q_stride=self.q_stride,
                            kv=b2.KVLayout(p(d["k"]), p(d["v"]), p(d["table"]), self.page, self.pps, self.hkv, self.hd),
                            pool_pages=self.pool_pages, row_start=p(d["start"]), ctx_len=p(d["ctx"]), tree=p(d.get("tree")),
                            max_ctx=int(max(1, (self.ctx + self.new).max())), ctx=p(d["out"]), ctx_stride=self.h * self.hd + 4,
                            err=p(d["err"]))
        for k, v in over.items():
            setattr(a, k, v)
        need = b2.lib().b2_attn_rows_scratch_bytes(a)
        self.d["scratch"] = torch.full((need + 16,), 0x7F, dtype=torch.uint8, device="cuda")
        a.scratch, a.scratch_bytes = p(self.d["scratch"]), need
        return a

    def run(self, b2, **over):
        a = self.args(b2, **over)
        assert b2.lib().b2_attn_rows(a, None) == 0
        self.torch.cuda.synchronize()
        out = self.d["out"].cpu().numpy()
        assert (out[self.rows:] == 7.25).all() and (out[:, self.h * self.hd:] == 7.25).all()
        return out[:self.rows, :self.h * self.hd].reshape(self.rows, self.h, self.hd).astype(np.float64), int(self.d["err"].item())

    def check(self, b2, **over):
        got, err = self.run(b2, **over)
        assert err == 0
        top = np.nanmax(np.abs(self.v)) if np.isfinite(self.v).any() else 1.0
        assert np.isfinite(got).all()
        assert np.abs(got - self.reference()).max(initial=0) <= ATTN_TOL * top


SHAPES = [(32, 8, 128, 64), (9, 3, 64, 64), (6, 6, 48, 16), (8, 1, 128, 24), (4, 2, 16, 7), (5, 1, 80, 128), (16, 2, 112, 1),
          (1, 1, 128, 64), (24, 1, 32, 33)]


@pytest.mark.parametrize("h,hkv,hd,page", SHAPES)
def test_attn_tree_shapes(b2, torch, h, hkv, hd, page):
    Scene(torch, h, hkv, hd, page, [70, 0, 129, 5], [8, 3, 1, 17], seed=hd).check(b2)


@pytest.mark.parametrize("new", [1, 2, 31, 32, 33, 63, 64])
def test_attn_tree_sizes(b2, torch, new):
    Scene(torch, 8, 2, 64, 64, [100], [new], seed=new).check(b2)


@pytest.mark.parametrize("ctx", [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 200, 1000])
def test_attn_tree_context_lengths(b2, torch, ctx):
    Scene(torch, 4, 1, 128, 64, [ctx], [9], seed=ctx).check(b2)


@pytest.mark.parametrize("ctx,new", [(0, 1), (0, 5), (0, 64), (3, 65), (190, 130), (64, 128), (1000, 300)])
@pytest.mark.parametrize("h,hkv,hd", [(8, 2, 128), (3, 3, 64)])
def test_attn_chain(b2, torch, h, hkv, hd, ctx, new):
    Scene(torch, h, hkv, hd, 64, [ctx], [new], tree=False, seed=ctx + new).check(b2)


def test_attn_ragged_batch_with_empty_items(b2, torch):
    Scene(torch, 8, 2, 128, 64, [500, 40, 0, 1200, 64, 7], [4, 0, 6, 64, 0, 1], seed=3, q_pad=8).check(b2)
    Scene(torch, 8, 2, 64, 16, [500, 40, 0, 333], [400, 0, 70, 1], tree=False, seed=4).check(b2)


def test_attn_long_context_is_split(b2, torch):
    """One KV head, 9000 places: the range is split over CTAs and joined."""
    Scene(torch, 4, 1, 64, 64, [9000], [3], seed=8).check(b2)


def test_attn_many_items(b2, torch):
    n = 150
    rng = np.random.default_rng(5)
    Scene(torch, 2, 1, 64, 32, rng.integers(0, 90, n), rng.integers(0, 7, n), seed=6).check(b2)


def test_attn_large_scores(b2, torch):
    """Scores of +-60 (one weight takes all) and keys of very different sizes."""
    s = Scene(torch, 4, 2, 64, 16, [50], [6], seed=9)
    got, err = s.run(b2)
    assert err == 0
    s.q *= 0.02
    s.k *= 100.0
    a, err = s.run(b2)
    assert err == 0 and np.isfinite(a).all()
    top = np.nanmax(np.abs(s.v))
    assert np.abs(a - s.reference()).max() <= ATTN_TOL * top


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60])
def test_attn_value_scale(b2, torch, scale):
    """V times a power of two gives the outputs times it, bit for bit."""
    s = Scene(torch, 4, 2, 64, 16, [80], [6], seed=10)
    a, err = s.run(b2)
    s.v *= np.float32(scale)
    b, err2 = s.run(b2)
    assert err == 0 and err2 == 0
    assert (a.astype(np.float32) * np.float32(scale) == b.astype(np.float32)).all()


def test_attn_keys_of_mixed_sizes(b2, torch):
    """Values of one place far larger than the others', at a place of little weight."""
    s = Scene(torch, 2, 1, 64, 16, [40], [4], seed=12)
    pg, off = s.place(0, 11)
    s.v[pg, :, off] *= 1e4
    got, err = s.run(b2)
    assert err == 0
    ref = s.reference()
    # the bound holds per place: sum_j |dp_j| |v_j|, with the large place's own weight
    assert np.abs(got - ref).max() <= ATTN_TOL * (4.0 + np.abs(ref).max())


def test_attn_masked_places_may_hold_anything(b2, torch):
    """A NaN or infinity in a drafted row's K or V reaches the rows that see it and no other."""
    for bad in (np.nan, np.inf, -np.inf):
        for which in ("k", "v"):
            s = Scene(torch, 4, 2, 64, 16, [37], [10], seed=13)
            ref = s.reference()
            victim = 6
            pg, off = s.place(0, 37 + victim)
            getattr(s, which)[pg, 1, off, 5] = bad
            got, err = s.run(b2)
            for i in range(10):
                hit = bool(s.masks[i] >> victim & 1)
                assert np.isnan(got[i, 2:]).all() == hit
                if not hit:
                    assert np.abs(got[i, 2:] - ref[i, 2:]).max() <= ATTN_TOL * 5
                assert np.abs(got[i, :2] - ref[i, :2]).max() <= ATTN_TOL * 5
            assert err == ERR_NONFINITE


@pytest.mark.parametrize("big", [3e3, 1e10, 1e30, 3e38])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("h,hkv,hd,new,victim", [(4, 2, 64, 10, 6), (2, 1, 128, 16, 3), (8, 2, 128, 24, 17), (4, 1, 64, 40, 9)])
def test_attn_hidden_place_takes_no_precision(b2, torch, h, hkv, hd, new, victim, which, big):
    """A finite K or V of any size in a drafted row: the rows that do not see it keep their error bound."""
    s = Scene(torch, h, hkv, hd, 16, [37], [new], seed=13)
    ref = s.reference()
    pg, off = s.place(0, 37 + victim)
    getattr(s, which)[pg, :, off] = big * np.sign(getattr(s, which)[pg, :, off])
    got, err = s.run(b2)
    for i in range(new):
        if not s.masks[i] >> victim & 1:
            assert np.abs(got[i] - ref[i]).max() <= ATTN_TOL * 5


@pytest.mark.parametrize("h,hkv,hd,new", [(4, 2, 64, 10), (8, 2, 128, 24)])
@pytest.mark.parametrize("at", [5, 20, 36])
def test_attn_place_of_no_weight_takes_no_precision(b2, torch, h, hkv, hd, new, at):
    """A cached place whose K is 2^14 times the others' in one direction: rows it draws to itself give its V,
    the others do as if it were not there, also where its V is 2^40."""
    s = Scene(torch, h, hkv, hd, 16, [37], [new], seed=16)
    pg, off = s.place(0, at)
    s.k[pg, :, off] = 0
    s.k[pg, :, off, 3] = 2.0 ** 14
    s.v[pg, :, off] = 2.0 ** 40
    q = s.q[:s.rows, :h * hd].reshape(s.rows, h, hd)
    q[:, :, 3] = np.where(q[:, :, 3] > 0, 1, -1)  # scores of +-2^14 / sqrt(hd)
    got, err = s.run(b2)
    assert err == 0
    drawn = q[:, :, 3] > 0
    assert drawn.any() and not drawn.all()
    assert (np.abs(got[drawn] - 2.0 ** 40) <= ATTN_TOL * 2.0 ** 40).all()
    t = 37 + new
    pages, offs = s.table[0, np.arange(t) // 16], np.arange(t) % 16
    for i in range(new):
        seen = [x for x in s.sees(0, i) if x != at]
        for hh in range(h):
            if drawn[i, hh]:
                continue
            K = s.k[pages[seen], hh // (h // hkv), offs[seen]].astype(np.float64)
            V = s.v[pages[seen], hh // (h // hkv), offs[seen]].astype(np.float64)
            w = np.exp((sc := K @ q[i, hh].astype(np.float64) / np.sqrt(hd)) - sc.max())
            assert np.abs(got[i, hh] - w @ V / w.sum()).max() <= ATTN_TOL * 5


@pytest.mark.parametrize("h,hkv,hd,new", [(4, 2, 64, 10), (2, 1, 128, 16), (8, 2, 128, 40), (4, 1, 48, 64)])
def test_attn_values_of_mixed_sizes(b2, torch, h, hkv, hd, new):
    """Every place's V times a power of two of its own, 2^-14 to 2^14."""
    s = Scene(torch, h, hkv, hd, 16, [150], [new], seed=18)
    s.v *= np.ldexp(np.float32(1), np.random.default_rng(7).integers(-14, 15, s.v.shape[0] * 16)).reshape(-1, 1, 16, 1).astype(np.float32)
    got, err = s.run(b2)
    assert err == 0
    ref, v = s.reference(), s.v
    s.v = np.abs(v)
    size = s.reference()  # sum_j p_j |v_j|, per dimension
    # a product keeps 2^-22 of itself, an element of V 2^-25 of 1 besides (where no place of 2^12 is near)
    assert (np.abs(got - ref) <= ATTN_TOL * size.max(-1, keepdims=True) + 2.0 ** -24).all()


def test_attn_nonfinite_query(b2, torch):
    s = Scene(torch, 4, 2, 64, 16, [37], [5], seed=14)
    ref = s.reference()
    s.q[2, 64 + 3] = np.inf
    got, err = s.run(b2)
    assert err == ERR_NONFINITE and np.isnan(got[2, 1]).all()
    got[2, 1] = ref[2, 1]
    assert np.abs(got - ref).max() <= ATTN_TOL * 5


def test_attn_row_that_sees_nothing(b2, torch):
    s = Scene(torch, 4, 2, 64, 16, [0, 5], [4, 3], seed=15)
    s.masks[2] = 0
    got, err = s.run(b2)
    assert err == 0 and (got[2] == 0).all()
    assert np.abs(got - s.reference()).max() <= ATTN_TOL * 5


def test_attn_lengths_that_do_not_fit(b2, torch):
    """The item's rows stay as they were; the others are computed."""
    s = Scene(torch, 4, 2, 64, 16, [20, 9], [4, 3], seed=16)
    ref = s.reference()
    s.ctx = np.array([20, 100])
    got, err = s.run(b2, max_ctx=24)
    assert err == ERR_POSITION and (got[4:] == 7.25).all()
    assert np.abs(got[:4] - ref[:4]).max() <= ATTN_TOL * 5
    s.ctx = np.array([-1, 9])
    got, err = s.run(b2, max_ctx=24)
    assert err == ERR_POSITION and (got[:4] == 7.25).all()
    assert np.abs(got[4:] - ref[4:]).max() <= ATTN_TOL * 5
    s.ctx = np.array([20, 9])
    got, err = s.run(b2, max_rows=3)
    assert err == ERR_POSITION and (got[:4] == 7.25).all()


@pytest.mark.parametrize("page_id", [-3, 1 << 20])
def test_attn_bad_page(b2, torch, page_id):
    """A page id outside the pool is reported and its places are not seen."""
    s = Scene(torch, 4, 2, 64, 16, [40], [3], seed=17)
    s.table[0, 1] = page_id
    got, err = s.run(b2)
    assert err == ERR_POSITION
    keep = s.sees
    s.sees = lambda b, i: [j for j in keep(b, i) if j // 16 != 1]
    s.table[0, 1] = 0
    s.k, s.v = np.nan_to_num(s.k), np.nan_to_num(s.v)
    assert np.abs(got - s.reference()).max() <= ATTN_TOL * 5


def test_attn_same_bits_every_time(b2, torch):
    s = Scene(torch, 8, 2, 128, 64, [3000, 100], [12, 40], seed=18)
    a, _ = s.run(b2)
    for _ in range(3):
        b, _ = s.run(b2)
        assert (a == b).all()


def test_attn_pool_past_32_bits(b2, torch):
    """Pages whose element offsets pass 2^32 (pools of 17 GB each)."""
    hkv, page, hd = 8, 64, 128
    n = (1 << 32) // (hkv * page * hd) + 40
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("not enough device memory free")
    s = Scene(torch, 8, hkv, hd, page, [150], [5], seed=19)
    a = s.args(b2)
    table = np.full_like(s.table, -1)
    ids = [n - 1, 3, n - 20]
    table[0, :3] = ids
    k, v = (torch.empty(n, hkv, page, hd, device="cuda") for _ in range(2))
    for i, pg in enumerate(ids):
        k[pg], v[pg] = s.d["k"][int(s.table[0, i])], s.d["v"][int(s.table[0, i])]
    td = dev(torch, table)
    a.kv.k_pool, a.kv.v_pool, a.kv.page_table, a.pool_pages = p(k), p(v), p(td), n
    assert b2.lib().b2_attn_rows(a, None) == 0
    torch.cuda.synchronize()
    got = s.d["out"].cpu().numpy()[:5, :8 * hd].reshape(5, 8, hd)
    assert int(s.d["err"].item()) == 0
    assert np.abs(got - s.reference()).max() <= ATTN_TOL * 5


@pytest.mark.parametrize("new", [15, 16, 17, 127, 128, 129, 384, 385])
@pytest.mark.parametrize("hd", [64, 128])
def test_attn_row_counts(b2, torch, hd, new):
    """Around the numbers of rows at which another kernel or block starts."""
    Scene(torch, 1, 1, hd, 64, [300], [new], tree=new <= 64, seed=new).check(b2)


@pytest.mark.parametrize("ctx", [2046, 2047, 2048])
def test_attn_one_token_at_long_contexts(b2, torch, ctx):
    Scene(torch, 4, 1, 64, 64, [ctx, 1, 17, 0, 1000], [1, 1, 1, 1, 1], seed=ctx).check(b2)
    Scene(torch, 4, 4, 128, 64, [ctx, 130], [2, 1], seed=ctx).check(b2)


@pytest.mark.parametrize("h,hkv,hd", [(16, 2, 128), (8, 1, 64), (16, 2, 80), (10, 1, 32)])
@pytest.mark.parametrize("ctx", [[0], [1], [64, 127], [128, 0, 500], [2500]])
def test_attn_many_rows_of_trees(b2, torch, h, hkv, hd, ctx):
    """Four blocks of 128 rows and more share an item's K and V."""
    Scene(torch, h, hkv, hd, 16, ctx, [64] + [41, 0, 9][:len(ctx) - 1], seed=h + hd).check(b2)


def test_attn_many_rows_of_ragged_chunks(b2, torch):
    Scene(torch, 8, 2, 128, 24, [500, 40, 0, 1, 63], [400, 0, 129, 1, 65], tree=False, seed=30, q_pad=4).check(b2)
    Scene(torch, 4, 1, 64, 64, [3000], [130], tree=False, seed=31).check(b2)


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38, 1e10])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("victim", [3, 40])
def test_attn_many_rows_masked_places(b2, torch, which, bad, victim):
    s = Scene(torch, 8, 1, 128, 16, [90], [64], seed=32)
    ref = s.reference()
    pg, off = s.place(0, 90 + victim)
    getattr(s, which)[pg, :, off] = bad
    got, err = s.run(b2)
    hits = 0
    for i in range(64):
        if s.masks[i] >> victim & 1:
            hits += 1
            if not np.isfinite(bad):
                assert np.isnan(got[i]).all()
        else:
            assert np.abs(got[i] - ref[i]).max() <= ATTN_TOL * 5
    assert hits > 0 and (np.isfinite(bad) or err == ERR_NONFINITE)


def test_attn_many_rows_of_mixed_sizes(b2, torch):
    s = Scene(torch, 8, 1, 128, 16, [300], [64], seed=33)
    s.v *= np.ldexp(np.float32(1), np.random.default_rng(8).integers(-14, 15, s.v.shape[0] * 16)).reshape(-1, 1, 16, 1).astype(np.float32)
    got, err = s.run(b2)
    assert err == 0
    ref, s.v = s.reference(), np.abs(s.v)
    assert (np.abs(got - ref) <= ATTN_TOL * s.reference().max(-1, keepdims=True) + 2.0 ** -24).all()


def test_attn_many_rows_refused_items_and_pages(b2, torch):
    s = Scene(torch, 8, 1, 64, 16, [200, 30], [64, 5], seed=34)
    s.table[0, 2] = -1
    s.q[s.start[1] + 1, 3] = np.nan
    got, err = s.run(b2)
    assert err == ERR_POSITION | ERR_NONFINITE
    keep = s.sees
    s.sees = lambda b, i: [j for j in keep(b, i) if b or j // 16 != 2]
    s.table[0, 2] = 0
    s.k, s.v, s.q = np.nan_to_num(s.k), np.nan_to_num(s.v), np.nan_to_num(s.q)
    ref = s.reference()
    assert np.isnan(got[s.start[1] + 1, 0]).all()
    got[s.start[1] + 1, 0] = ref[s.start[1] + 1, 0]
    assert np.abs(got - ref).max() <= ATTN_TOL * 5
    s.ctx = np.array([200, 900])
    got, err = s.run(b2, max_ctx=264)
    assert err == ERR_POSITION and (got[64:] == 7.25).all()


def test_attn_many_rows_without_room_for_operands(b2, torch):
    """A bound on the places so large that K and V are not laid out in scratch gives the same within both bounds."""
    s = Scene(torch, 8, 1, 128, 64, [150], [64], seed=35)
    ref = s.reference()
    a = s.args(b2)
    small = a.scratch_bytes
    s.pps = 9000
    wide = np.full((1, s.pps), -7, np.int32)
    wide[:, :s.table.shape[1]] = s.table
    s.table = wide
    a = s.args(b2, max_ctx=64 * 9000)
    assert 0 < small < 1 << 20 and a.scratch_bytes < 512 << 20
    assert b2.lib().b2_attn_rows(a, None) == 0
    torch.cuda.synchronize()
    got = s.d["out"].cpu().numpy()[:s.rows, :8 * 128].reshape(s.rows, 8, 128)
    assert int(s.d["err"].item()) == 0 and np.abs(got - ref).max() <= ATTN_TOL * 5


def test_attn_many_rows_graph_and_streams(b2, torch):
    """Captured and replayed with other lengths; calls at once with scratch of their own; the same bits each time."""
    s = Scene(torch, 8, 1, 128, 64, [900, 30], [64, 50], seed=36)
    t = Scene(torch, 8, 1, 64, 64, [300, 500], [60, 64], seed=37)
    a, b = s.args(b2), t.args(b2)
    st, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    b2.check("warm", b2.lib().b2_attn_rows(a, st.cuda_stream))
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        b2.check("capture", b2.lib().b2_attn_rows(a, torch.cuda.current_stream().cuda_stream))
    first = None
    for ctx in ([900, 30], [100, 11], [900, 30]):
        s.ctx = np.array(ctx)
        s.k, s.v = np.nan_to_num(s.k), np.nan_to_num(s.v)
        s.table = np.abs(s.table) % s.pool_pages
        for name, x in (("k", s.k), ("v", s.v), ("table", s.table), ("ctx", s.ctx.astype(np.int32))):
            s.d[name].copy_(dev(torch, x))
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(st):
                g.replay()
            b2.check("beside", b2.lib().b2_attn_rows(b, s2.cuda_stream))
        torch.cuda.synchronize()
        got = s.d["out"].cpu().numpy()[:s.rows, :8 * 128].reshape(s.rows, 8, 128)
        assert np.abs(got - s.reference()).max() <= ATTN_TOL * 5
        if ctx == [900, 30]:
            assert first is None or (got == first).all()
            first = got
    got = t.d["out"].cpu().numpy()[:t.rows, :8 * 64].reshape(t.rows, 8, 64)
    assert np.abs(got - t.reference()).max() <= ATTN_TOL * 5


def test_attn_matches_single_query_attention(b2, torch):
    """One row per item is b2_attn's case: the same numbers within both bounds."""
    s = Scene(torch, 8, 2, 128, 64, [300, 77, 0], [1, 1, 1], seed=20)
    got, err = s.run(b2)
    L, d = b2.lib(), s.d
    pos = dev(torch, s.ctx, np.int32)
    out = torch.zeros(3, 8 * 128, device="cuda")
    qd = dev(torch, s.q[:3, :8 * 128])
    kv = b2.KVLayout(p(d["k"]), p(d["v"]), p(d["table"]), 64, s.pps, 2, 128)
    a = b2.AttnArgs(batch=3, n_heads=8, n_kv_heads=2, head_dim=128, q=p(qd), kv=kv, positions=p(pos), max_ctx=s.pps * 64,
                    ctx=p(out), err=p(d["err"]))
    sc = torch.zeros(L.b2_attn_scratch_bytes(a), dtype=torch.uint8, device="cuda")
    cn = torch.zeros(L.b2_attn_counters_len(a), dtype=torch.int32, device="cuda")
    a.scratch, a.scratch_bytes, a.counters, a.counters_len = p(sc), sc.numel(), p(cn), cn.numel()
    assert L.b2_attn(a, None) == 0
    torch.cuda.synchronize()
    assert np.abs(out.cpu().numpy().reshape(3, 8, 128) - got).max() <= 2 * ATTN_TOL * 5


def test_attn_graph_replay_and_two_streams(b2, torch):
    """Captured once, replayed with other lengths; two calls at once with scratch of their own."""
    s = Scene(torch, 8, 2, 64, 64, [900, 30], [6, 20], seed=21)
    a = s.args(b2)
    st = torch.cuda.Stream()
    b2.check("warm", b2.lib().b2_attn_rows(a, st.cuda_stream))
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        b2.check("capture", b2.lib().b2_attn_rows(a, torch.cuda.current_stream().cuda_stream))
    for ctx in ([900, 30], [100, 11], [0, 33]):
        s.ctx = np.array(ctx)
        s.k, s.v = np.nan_to_num(s.k), np.nan_to_num(s.v)
        s.d["k"].copy_(dev(torch, s.k))
        s.d["v"].copy_(dev(torch, s.v))
        s.table = np.abs(s.table) % s.pool_pages
        s.d["table"].copy_(dev(torch, s.table))
        s.d["ctx"].copy_(dev(torch, s.ctx, np.int32))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = s.d["out"].cpu().numpy()[:s.rows, :8 * 64].reshape(s.rows, 8, 64)
        assert np.abs(got - s.reference()).max() <= ATTN_TOL * 5
    t = Scene(torch, 8, 2, 64, 64, [700, 300], [6, 20], seed=22)
    b = t.args(b2)
    torch.cuda.synchronize()
    s2 = torch.cuda.Stream()
    for _ in range(20):
        b2.check("one", b2.lib().b2_attn_rows(a, st.cuda_stream))
        b2.check("two", b2.lib().b2_attn_rows(b, s2.cuda_stream))
    torch.cuda.synchronize()
    for x in (s, t):
        got = x.d["out"].cpu().numpy()[:x.rows, :8 * 64].reshape(x.rows, 8, 64)
        assert np.abs(got - x.reference()).max() <= ATTN_TOL * 5


# ---- b2_kv_plan ---------------------------------------------------------------------------------------


def plan_case(torch, ctx, new, page, tree, seed=0, spare=5, slack=1):
    rng = np.random.default_rng(seed)
    ctx, new = np.array(ctx), np.array(new)
    have = -(-ctx // page)
    pps = int(max(1, (-(-(ctx + new) // page)).max())) + slack
    pool = int(have.sum() + (-(-new // page) + 1).sum()) + 4
    order = rng.permutation(pool).astype(np.int32)
    table = np.full((len(ctx), pps), -9, np.int32)
    at = 0
    for b, u in enumerate(have):
        table[b, :u] = order[at:at + u]
        at += u
    masks = [m for t in new for m in make_tree(int(t), rng)[1]] if tree else None
    return dict(ctx=ctx, new=new, page=page, pps=pps, pool=pool, table=table, mapped=have, free=order[at:], masks=masks, spare=spare)


def plan_run(b2, torch, c, max_rows=None, **over):
    rows = int(c["new"].sum())
    cap = rows + c["spare"] if max_rows is None else max_rows
    d = dict(ctx=dev(torch, c["ctx"], np.int32), new=dev(torch, c["new"], np.int32), mapped=dev(torch, c["mapped"], np.int32),
             free=dev(torch, c["free"], np.int32), count=dev(torch, [len(c["free"])], np.int32), table=dev(torch, c["table"]),
             mo=dev(torch, np.full(len(c["ctx"]), -2), np.int32), fo=dev(torch, [-2], np.int32),
             start=dev(torch, np.full(len(c["ctx"]) + 1, -2), np.int32), err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    for k in ("item", "pos", "slot"):
        d[k] = torch.full((max(cap, 1),), -2, dtype=torch.int32, device="cuda")
    if c["masks"] is not None:
        d["tree"] = dev(torch, np.array(list(c["masks"]) + [0] * 64, np.uint64).view(np.int64))
    a = b2.KvPlanArgs(batch=len(c["ctx"]), max_rows=cap, page_tokens=c["page"], pages_per_seq=c["pps"], pool_pages=c["pool"],
                      ctx_len=p(d["ctx"]), new_len=p(d["new"]), tree=p(d.get("tree")), mapped=p(d["mapped"]), free_pages=p(d["free"]),
                      free_count=p(d["count"]), page_table=p(d["table"]), mapped_out=p(d["mo"]), free_out=p(d["fo"]),
                      row_start=p(d["start"]), row_item=p(d["item"]), row_pos=p(d["pos"]), row_slot=p(d["slot"]), err=p(d["err"]))
    for k, v in over.items():
        setattr(a, k, v)
    assert b2.lib().b2_kv_plan(a, None) == 0
    torch.cuda.synchronize()
    return {k: t.cpu().numpy() for k, t in d.items()}


def plan_check(b2, torch, c):
    got = plan_run(b2, torch, c)
    rows, free = int(c["new"].sum()), list(c["free"])
    table, item, pos, slot, start, mapped = c["table"].copy(), [], [], [], [0], []
    for b, (cx, n) in enumerate(zip(c["ctx"], c["new"])):
        need = max(int(c["mapped"][b]), -(-int(cx + n) // c["page"]))
        for lp in range(int(c["mapped"][b]), need):
            table[b, lp] = free.pop()
        mapped.append(need)
        for i in range(int(n)):
            depth = bin(c["masks"][start[-1] + i]).count("1") - 1 if c["masks"] is not None else i
            at = int(cx) + i
            item.append(b)
            pos.append(int(cx) + depth)
            slot.append(int(table[b, at // c["page"]]) * c["page"] + at % c["page"])
        start.append(start[-1] + int(n))
    assert got["err"][0] == 0
    assert (got["start"] == start).all() and (got["mo"] == mapped).all() and got["fo"][0] == len(free)
    assert (got["table"] == table).all()
    for k, want in (("item", item), ("pos", pos), ("slot", slot)):
        assert (got[k][:rows] == want).all() and (got[k][rows:] == -2).all()


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("tree", [True, False])
def test_plan_small(b2, torch, page, tree):
    plan_check(b2, torch, plan_case(torch, [0, 5, 64, 63, 100, 0], [3, 1, 0, 64, 17, 0], page, tree, seed=page))


def test_plan_one_token(b2, torch):
    plan_check(b2, torch, plan_case(torch, [64], [1], 64, True))
    plan_check(b2, torch, plan_case(torch, [0], [1], 64, False))
    plan_check(b2, torch, plan_case(torch, [10], [0], 64, False))


@pytest.mark.parametrize("batch", [31, 512, 513, 2000, 4096])
def test_plan_batches(b2, torch, batch):
    rng = np.random.default_rng(batch)
    plan_check(b2, torch, plan_case(torch, rng.integers(0, 300, batch), rng.integers(0, 40, batch), 16, batch % 2 == 0, seed=batch))


def test_plan_long_chunks(b2, torch):
    plan_check(b2, torch, plan_case(torch, [5000, 0, 77], [20000, 1, 9000], 64, False))


def test_plan_pages_held_ahead(b2, torch):
    """A sequence that already holds more pages than it needs keeps them."""
    c = plan_case(torch, [10, 20], [4, 30], 16, False, slack=4)
    c["mapped"] = np.array([4, 2])
    c["table"][0, 1:4] = [c["free"][0], c["free"][1], c["free"][2]]
    c["free"] = c["free"][3:]
    plan_check(b2, torch, c)


def plan_refused(b2, torch, c, bit, **over):
    got = plan_run(b2, torch, c, **over)
    assert got["err"][0] == bit
    assert (got["start"] == 0).all() and (got["mo"] == c["mapped"]).all() and got["fo"][0] == len(c["free"])
    assert (got["table"] == c["table"]).all()
    for k in ("item", "pos", "slot"):
        assert (got[k] == -2).all()


def test_plan_steps_that_do_not_fit(b2, torch):
    def case(ctx=(10, 20), new=(4, 30)):
        return plan_case(torch, list(ctx), list(new), 16, False)
    plan_refused(b2, torch, case(), ERR_CAPACITY, max_rows=33)
    c = case()
    c["free"] = c["free"][:1]
    plan_refused(b2, torch, c, ERR_CAPACITY)
    c = case()
    c["new"] = np.array([4, 1000])
    plan_refused(b2, torch, c, ERR_POSITION, max_rows=2000)
    for ctx, new in (((-1, 20), (4, 3)), ((10, 20), (4, -1)), ((2 ** 31 - 1, 20), (4, 3)), ((10, 20), (2 ** 31 - 1, 3))):
        c = case()
        c["ctx"], c["new"] = np.array(ctx), np.array(new)
        c["spare"] = 100 - int(c["new"].sum())
        plan_refused(b2, torch, c, ERR_POSITION, max_rows=100)
    c = case()
    c["mapped"] = np.array([0, 2])   # ten cached tokens on no page
    plan_refused(b2, torch, c, ERR_POSITION)
    c = plan_case(torch, [3], [65], 16, False)
    c["masks"] = [1] * 65
    plan_refused(b2, torch, c, ERR_POSITION)


def test_plan_bad_page(b2, torch):
    c = plan_case(torch, [20, 3], [4, 4], 16, False)
    c["table"][0, 1] = c["pool"]
    got = plan_run(b2, torch, c)
    assert got["err"][0] == ERR_POSITION
    assert (got["slot"][:4] == -1).all() and (got["slot"][4:8] >= 0).all()


# ---- b2_rows_append ------------------------------------------------------------------------------------


def append_run(b2, torch, h, hkv, hd, page, m, seed=0, live=None, rope=True, slots=None, positions=None, pad=0):
    rng = np.random.default_rng(seed)
    pages = -(-m // page) + 2
    y = rng.normal(0, 1, (m, (h + 2 * hkv) * hd + pad)).astype(np.float32)
    pos = rng.integers(0, 100000, m) if positions is None else np.array(positions)
    slots = rng.permutation(pages * page)[:m] if slots is None else np.array(slots)
    k0, v0 = (rng.normal(0, 1, (pages, hkv, page, hd)).astype(np.float32) for _ in range(2))
    freq = (1.0 / np.power(np.float32(500000.0), np.arange(0, hd, 2, dtype=np.float32) / np.float32(hd))).astype(np.float32)
    d = dict(y=dev(torch, y), pos=dev(torch, pos, np.int32), slots=dev(torch, slots, np.int32), k=dev(torch, k0), v=dev(torch, v0),
             freq=dev(torch, freq), q=torch.full((m, h * hd + 4), 7.25, device="cuda"), err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if live is not None:
        d["live"] = dev(torch, [live], np.int32)
    a = b2.RowsAppendArgs(m=m, y=p(d["y"]), y_stride=y.shape[1], q_rows=h * hd, q=p(d["q"]), q_stride=h * hd + 4,
                          rope_freq=p(d["freq"]) if rope else None, positions=p(d["pos"]) if rope else None, slots=p(d["slots"]),
                          n_rows=p(d.get("live")), kv=b2.KVLayout(p(d["k"]), p(d["v"]), None, page, 0, hkv, hd), pool_pages=pages,
                          err=p(d["err"]))
    assert b2.lib().b2_rows_append(a, None) == 0
    torch.cuda.synchronize()
    # float64 form of the rotation at the f32 angle
    rows = y[:, :(h + 2 * hkv) * hd].astype(np.float64).reshape(m, h + 2 * hkv, hd)
    if rope:
        ang = (pos.astype(np.float32)[:, None] * freq[None]).astype(np.float64)[:, None]
        x0, x1 = rows[:, :h + hkv, 0::2].copy(), rows[:, :h + hkv, 1::2].copy()
        rows[:, :h + hkv, 0::2] = x0 * np.cos(ang) - x1 * np.sin(ang)
        rows[:, :h + hkv, 1::2] = x0 * np.sin(ang) + x1 * np.cos(ang)
    n = m if live is None else min(max(live, 0), m)
    q, k, v = np.full((m, h * hd), 7.25), k0.astype(np.float64), v0.astype(np.float64)
    for i in range(n):
        if rope and pos[i] < 0:
            continue
        q[i] = rows[i, :h].reshape(-1)
        if 0 <= slots[i] < pages * page:
            k[slots[i] // page, :, slots[i] % page] = rows[i, h:h + hkv]
            v[slots[i] // page, :, slots[i] % page] = rows[i, h + hkv:]
    tol = 2.0 ** -21 * np.abs(y).max()
    got_q = d["q"].cpu().numpy()
    assert (got_q[:, h * hd:] == 7.25).all()
    for got, want in ((got_q[:, :h * hd], q), (d["k"].cpu().numpy(), k), (d["v"].cpu().numpy(), v)):
        assert np.abs(got - want).max() <= tol
    assert (d["v"].cpu().numpy() == v.astype(np.float32)).all()
    return int(d["err"].item()), a, d


@pytest.mark.parametrize("h,hkv,hd,page", SHAPES)
@pytest.mark.parametrize("m", [1, 7, 150])
def test_append_shapes(b2, torch, h, hkv, hd, page, m):
    assert append_run(b2, torch, h, hkv, hd, page, m, seed=m, pad=4 * (m % 2))[0] == 0


@pytest.mark.parametrize("h,hkv,hd", [(2, 1, 1024), (3, 3, 516), (5, 1, 512), (150, 75, 16), (1, 1, 4)])
@pytest.mark.parametrize("m", [1, 40])
def test_append_head_sizes(b2, torch, h, hkv, hd, m):
    """Heads wider than a block's threads take, and more heads than a thread loads at a time."""
    assert append_run(b2, torch, h, hkv, hd, 16, m, seed=m)[0] == 0


def test_append_rows_in_use(b2, torch):
    for live in (0, 1, 5, 9, 40, -3):
        assert append_run(b2, torch, 4, 2, 64, 16, 9, live=live)[0] == 0


def test_append_without_rope(b2, torch):
    assert append_run(b2, torch, 4, 2, 64, 16, 9, rope=False)[0] == 0


def test_append_bad_rows(b2, torch):
    assert append_run(b2, torch, 4, 2, 64, 16, 4, slots=[3, -1, 5, -9])[0] == 0
    assert append_run(b2, torch, 4, 2, 64, 16, 4, slots=[3, 48, 5, 2 ** 31 - 1])[0] == ERR_POSITION
    assert append_run(b2, torch, 4, 2, 64, 16, 4, positions=[3, -1, 5, 0])[0] == ERR_POSITION


def test_append_same_bits_as_rows_epilogue(b2, torch):
    """Chain rows through b2_rows_epilogue (the decode path's own K/V append)."""
    h, hkv, hd, page, m = 8, 2, 64, 16, 20
    pos = np.arange(m) + 5
    perm = np.random.default_rng(3).permutation(4)[:2 + 1]
    slots = perm[pos // page] * page + pos % page
    _, a, d = append_run(b2, torch, h, hkv, hd, page, m, slots=slots, positions=pos)

    class RowsArgs(C.Structure):
        _fields_ = [("epilogue", C.c_uint32), ("m", C.c_uint32), ("y", C.c_void_p), ("y_stride", C.c_uint32), ("rows", C.c_uint32),
                    ("out", C.c_void_p), ("out_stride", C.c_uint32), ("q_rows", C.c_uint32), ("kv_rows", C.c_uint32),
                    ("rope_freq", C.c_void_p), ("positions", C.c_void_p), ("kv", b2.KVLayout), ("argmax", C.c_void_p),
                    ("row_offset", C.c_uint32), ("err", C.c_void_p), ("pdl", C.c_int)]
    table = dev(torch, np.tile(np.pad(perm, (0, 1))[None].astype(np.int32), (m, 1)))
    k, v, q = torch.zeros_like(d["k"]), torch.zeros_like(d["v"]), torch.zeros(m, h * hd, device="cuda")
    r = RowsArgs(epilogue=2, m=m, y=p(d["y"]), y_stride=a.y_stride, rows=(h + 2 * hkv) * hd, out=p(q), out_stride=h * hd, q_rows=h * hd,
                 kv_rows=hkv * hd, rope_freq=p(d["freq"]), positions=p(d["pos"]),
                 kv=b2.KVLayout(p(k), p(v), p(table), page, 4, hkv, hd), err=p(d["err"]))
    fn = b2.lib().b2_rows_epilogue
    fn.restype, fn.argtypes = C.c_int, [C.POINTER(RowsArgs), C.c_void_p]
    assert fn(r, None) == 0
    torch.cuda.synchronize()
    assert (q.cpu().numpy() == d["q"].cpu().numpy()[:, :h * hd]).all()
    for i in range(m):
        for mine, theirs in ((d["k"], k), (d["v"], v)):
            assert (mine[slots[i] // page, :, slots[i] % page] == theirs[slots[i] // page, :, slots[i] % page]).all()


# ---- b2_tree_accept, b2_kv_compact --------------------------------------------------------------------


def accept_reference(parents, tokens, nxt):
    path, cur = ([0], 0) if parents else ([], 0)
    while path:
        child = [i for i in range(1, len(parents)) if parents[i] == cur and tokens[i] == nxt[cur]]
        if not child:
            break
        cur = child[0]
        path.append(cur)
    return path, (nxt[cur] if path else 0xFFFFFFFF)


def accept_run(b2, torch, start, tokens, masks, nxt, ctx, rows=None, max_rows=64):
    n = len(start) - 1
    keys = [(0xC0000000 << 32) | (0xFFFFFFFF - int(t)) for t in nxt]
    d = dict(start=dev(torch, start, np.int32), tokens=dev(torch, np.array(list(tokens) + [0], np.uint32).view(np.int32)),
             keys=dev(torch, np.array(keys + [0], np.uint64).view(np.int64)), ctx=dev(torch, ctx, np.int32),
             path=torch.full((n, 64), -5, dtype=torch.int32, device="cuda"), err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    for k in ("count", "next", "out"):
        d[k] = torch.full((n,), -5, dtype=torch.int32, device="cuda")
    if masks is not None:
        d["tree"] = dev(torch, np.array(list(masks) + [0], np.uint64).view(np.int64))
    a = b2.TreeAcceptArgs(batch=n, max_rows=max_rows, rows=len(tokens) if rows is None else rows, row_start=p(d["start"]), tokens=p(d["tokens"]),
                          tree=p(d.get("tree")), argmax=p(d["keys"]), ctx_len=p(d["ctx"]), path=p(d["path"]), count=p(d["count"]),
                          next=p(d["next"]), ctx_out=p(d["out"]), err=p(d["err"]))
    assert b2.lib().b2_tree_accept(a, None) == 0
    torch.cuda.synchronize()
    r = {k: t.cpu().numpy() for k, t in d.items()}
    r["next"] = r["next"].view(np.uint32)
    return r


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("vocab", [2, 3, 50])
def test_accept_random_trees(b2, torch, seed, vocab):
    """Small vocabularies, so branches go deep and siblings carry equal tokens."""
    rng = np.random.default_rng(seed)
    new = [0, 1, 64, 33, 32, 2] + [int(x) for x in rng.integers(0, 65, 9)]
    start = np.concatenate([[0], np.cumsum(new)])
    trees = [make_tree(n, rng) for n in new]
    tokens, nxt = rng.integers(0, vocab, start[-1]), rng.integers(0, vocab, start[-1])
    ctx = rng.integers(0, 1000, len(new))
    r = accept_run(b2, torch, start, tokens, [m for t in trees for m in t[1]], nxt, ctx)
    assert r["err"][0] == 0
    for b, (par, _) in enumerate(trees):
        path, follow = accept_reference(par if new[b] else [], tokens[start[b]:start[b + 1]], nxt[start[b]:start[b + 1]])
        assert r["count"][b] == len(path) and r["next"][b] == follow and r["out"][b] == ctx[b] + len(path)
        assert list(r["path"][b]) == path + [-1] * (64 - len(path))


def test_accept_chain(b2, torch):
    tokens = np.array([9, 1, 2, 3, 4] + list(range(64)))
    nxt = np.array([1, 2, 7, 4, 5] + list(range(1, 65)))
    r = accept_run(b2, torch, [0, 5, 69], tokens, None, nxt, [10, 0])
    assert list(r["count"]) == [3, 64] and list(r["next"]) == [7, 64] and list(r["out"]) == [13, 64]
    assert r["err"][0] == 0


def test_accept_large_token_ids(b2, torch):
    r = accept_run(b2, torch, [0, 2], [5, 4000000000], [1, 3], [4000000000, 4294967295], [0])
    assert r["count"][0] == 2 and r["next"][0] == 4294967295


def test_accept_bad_masks_and_lengths(b2, torch):
    r = accept_run(b2, torch, [0, 3], [0, 1, 1], [1, 1, 3 | 4], [1, 1, 8], [0])    # row 1 lacks its own bit, row 2 hangs off it
    assert r["err"][0] == ERR_TREE and r["count"][0] == 1 and r["next"][0] == 1
    r = accept_run(b2, torch, [0, 2], [0, 1], [1, 7], [1, 1], [0])                  # a bit past the row
    assert r["err"][0] == ERR_TREE and r["count"][0] == 1
    r = accept_run(b2, torch, [0, 2], [0, 1], [1, 2], [1, 1], [0])                  # no root
    assert r["err"][0] == ERR_TREE and r["count"][0] == 1
    r = accept_run(b2, torch, [0, 3], [0, 1, 1], [1, 3, 7], [1, 1, 8], [4], max_rows=2)
    assert r["err"][0] == ERR_POSITION and r["count"][0] == 0 and r["out"][0] == 4
    r = accept_run(b2, torch, [0, 3], [0, 1, 1], [1, 3, 7], [1, 1, 8], [4], rows=2)
    assert r["err"][0] == ERR_POSITION and r["count"][0] == 0


def compact_run(b2, torch, layers, hkv, hd, page, ctx, paths, pps=None, count=None, mutate=None, seed=0, pool_pages=None):
    rng = np.random.default_rng(seed)
    batch = len(ctx)
    pps = pps or max(1, max(-(-(c + 64) // page) for c in ctx))
    n = batch * pps + 2
    table = rng.permutation(n)[:batch * pps].reshape(batch, pps).astype(np.int32)
    if mutate is not None:
        mutate(table)
    k = rng.normal(0, 1, (layers, 2, n, hkv, page, hd)).astype(np.float32)
    kd, td, cd = dev(torch, k), dev(torch, table), dev(torch, ctx, np.int32)
    full = np.full((batch, 64), -1, np.int32)
    for b, path in enumerate(paths):
        full[b, :len(path)] = path
    pd, nd = dev(torch, full), dev(torch, [len(x) for x in paths] if count is None else count, np.int32)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kvs = (b2.KVLayout * layers)(*[b2.KVLayout(p(kd[i, 0]), p(kd[i, 1]), p(td), page, pps, hkv, hd) for i in range(layers)])
    a = b2.KvCompactArgs(n_layers=layers, layers=kvs, pool_pages=n if pool_pages is None else pool_pages, batch=batch, ctx_len=p(cd),
                         path=p(pd), count=p(nd), err=p(err))
    assert b2.lib().b2_kv_compact(a, None) == 0
    torch.cuda.synchronize()
    want = k.copy()
    for b, path in enumerate(paths):
        for i, j in enumerate(path):
            s, t = ctx[b] + j, ctx[b] + i
            if j < i or s // page >= pps or table[b, s // page] < 0 or table[b, s // page] >= n:
                continue
            want[:, :, table[b, t // page], :, t % page] = want[:, :, table[b, s // page], :, s % page]
    return kd.cpu().numpy(), want, int(err.item())


@pytest.mark.parametrize("layers,hkv,hd,page", [(2, 8, 128, 64), (30, 3, 64, 16), (1, 1, 16, 1), (70, 2, 48, 7), (3, 16, 112, 33)])
def test_compact(b2, torch, layers, hkv, hd, page):
    rng = np.random.default_rng(layers)
    paths = [[0], [], [0, 1, 2, 3], list(range(64)), sorted(rng.choice(np.arange(1, 64), 20, replace=False).tolist()),
             [0] + sorted(rng.choice(np.arange(1, 64), 7, replace=False).tolist()), [63]]
    paths[4] = [0] + paths[4]
    got, want, err = compact_run(b2, torch, layers, hkv, hd, page, [0, 5, 63, 64, 100, 31, 2], paths)
    assert err == 0 and (got == want).all()


def test_compact_pool_past_32_bits_of_places(b2, torch):
    """A pool of more than 2^32 places (69 GB of 16-byte rows; K and V the same)."""
    page, n = 1 << 16, (1 << 16) + 3
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough device memory free")
    pool = torch.empty(n, page, 4, device="cuda")
    table = dev(torch, [[n - 1, 2]], np.int32)
    rows = torch.arange(40, dtype=torch.float32, device="cuda").reshape(10, 4) + 1
    ctx = page - 3   # places page - 3 .. page + 6
    pool[n - 1, page - 3:] = rows[:3]
    pool[2, :7] = rows[3:]
    pool[2, page - 10:] = 0
    path = torch.full((1, 64), -1, dtype=torch.int32, device="cuda")
    path[0, :4] = dev(torch, [0, 2, 5, 9], np.int32)
    kv = (b2.KVLayout * 1)(b2.KVLayout(p(pool), p(pool), p(table), page, 2, 1, 4))
    d = dict(ctx=dev(torch, [ctx], np.int32), count=dev(torch, [4], np.int32), err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert b2.lib().b2_kv_compact(b2.KvCompactArgs(n_layers=1, layers=kv, pool_pages=n, batch=1, ctx_len=p(d["ctx"]), path=p(path),
                                                   count=p(d["count"]), err=p(d["err"])), None) == 0
    torch.cuda.synchronize()
    assert int(d["err"].item()) == 0
    assert (pool[n - 1, page - 3:] == rows[[0, 2, 5]]).all()
    assert (pool[2, 0] == rows[9]).all() and (pool[2, 1:7] == rows[4:]).all()


def test_compact_bad_rows(b2, torch):
    got, want, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [[0, 0, 5]])          # path below its index
    assert err == ERR_POSITION and (got == want).all()
    got, want, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [[0, 40]], pps=2)     # past the table row
    assert err == ERR_POSITION and (got == want).all()
    got, want, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [[]], count=[65])
    assert err == ERR_POSITION and (got == want).all()
    for page_id in (-4, 1 << 24):
        got, want, err = compact_run(b2, torch, 2, 2, 64, 16, [10], [[0, 9]], mutate=lambda t: t.__setitem__((0, 1), page_id))
        assert err == ERR_POSITION and (got == want).all()


# ---- the operators together ----------------------------------------------------------------------------


@pytest.mark.parametrize("h,hkv,hd", [(8, 1, 64), (4, 2, 128), (2, 2, 48)])
def test_steps_of_chunks(b2, torch, h, hkv, hd):
    """Three steps of prompt chunks over several layers that share one scratch, each kernel launched while
    the one before still runs: every row against float64."""
    batch, page, layers, pps = 3, 16, 5, 40
    rng = np.random.default_rng(hd)
    L = b2.lib()
    pool = batch * pps
    free = dev(torch, rng.permutation(pool), np.int32)
    ctx = torch.zeros(batch, dtype=torch.int32, device="cuda")
    mapped, count = torch.zeros_like(ctx), dev(torch, [pool], np.int32)
    table = torch.full((batch, pps), -1, dtype=torch.int32, device="cuda")
    k, v = (torch.full((layers, pool, hkv, page, hd), float("nan"), device="cuda") for _ in range(2))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    K, V = ([[np.zeros((0, hkv, hd))] * batch for _ in range(layers)] for _ in range(2))
    scratch = None
    for new in ([200, 0, 130], [1, 70, 260], [64, 3, 1]):
        rows, start = sum(new), np.concatenate([[0], np.cumsum(new)])
        nd = dev(torch, new, np.int32)
        d = {x: torch.full((rows,), -1, dtype=torch.int32, device="cuda") for x in ("item", "pos", "slot")}
        rs = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
        mo, fo = torch.zeros_like(mapped), torch.zeros_like(count)
        ys = rng.normal(0, 1, (layers, rows, (h + 2 * hkv) * hd)).astype(np.float32)
        y = dev(torch, ys)
        q, o = (torch.zeros(layers, rows, h * hd, device="cuda") for _ in range(2))
        kvs = [b2.KVLayout(p(k[l]), p(v[l]), p(table), page, pps, hkv, hd) for l in range(layers)]
        calls = [b2.AttnRowsArgs(batch=batch, n_heads=h, n_kv_heads=hkv, head_dim=hd, max_rows=max(new), rows=rows, q=p(q[l]),
                                 q_stride=h * hd, kv=kvs[l], pool_pages=pool, row_start=p(rs), ctx_len=p(ctx), max_ctx=pps * page,
                                 ctx=p(o[l]), ctx_stride=h * hd, err=p(err), pdl=1) for l in range(layers)]
        need = L.b2_attn_rows_scratch_bytes(calls[0])
        if scratch is None or scratch.numel() < need:
            scratch = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        b2.check("plan", L.b2_kv_plan(b2.KvPlanArgs(
            batch=batch, max_rows=rows, page_tokens=page, pages_per_seq=pps, pool_pages=pool, ctx_len=p(ctx), new_len=p(nd),
            mapped=p(mapped), free_pages=p(free), free_count=p(count), page_table=p(table), mapped_out=p(mo), free_out=p(fo),
            row_start=p(rs), row_item=p(d["item"]), row_pos=p(d["pos"]), row_slot=p(d["slot"]), err=p(err), pdl=1), None))
        for l, a in enumerate(calls):
            b2.check("append", L.b2_rows_append(b2.RowsAppendArgs(
                m=rows, y=p(y[l]), y_stride=y.shape[2], q_rows=h * hd, q=p(q[l]), q_stride=h * hd, slots=p(d["slot"]), kv=kvs[l],
                pool_pages=pool, err=p(err), pdl=1), None))
            a.scratch, a.scratch_bytes = p(scratch), scratch.numel()
            b2.check("attn", L.b2_attn_rows(a, None))
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        got = o.cpu().numpy().reshape(layers, rows, hkv, h // hkv, hd)
        yy = ys.astype(np.float64).reshape(layers, rows, h + 2 * hkv, hd)
        for l in range(layers):
            for b in range(batch):
                at = slice(start[b], start[b + 1])
                K[l][b] = np.concatenate([K[l][b], yy[l, at, h:h + hkv]])
                V[l][b] = np.concatenate([V[l][b], yy[l, at, h + hkv:]])
                if new[b] == 0:
                    continue
                t = len(K[l][b])
                s = np.einsum("nhgd,thd->nhgt", yy[l, at, :h].reshape(-1, hkv, h // hkv, hd), K[l][b]) / np.sqrt(hd)
                s = np.where((np.arange(t) <= t - new[b] + np.arange(new[b])[:, None])[:, None, None], s, -np.inf)
                w = np.exp(s - s.max(-1, keepdims=True))
                want = np.einsum("nhgt,thd->nhgd", w / w.sum(-1, keepdims=True), V[l][b])
                assert np.abs(got[l, at] - want).max() <= ATTN_TOL * 5
        ctx += nd
        mapped, count = mo, fo


def test_step_of_trees(b2, torch):
    """Two steps of ragged trees: plan, append, attention, verification and compaction; afterwards the
    cache holds what a plain replay of the taken tokens holds, and attention over it agrees."""
    h, hkv, hd, page, batch, layers = 8, 2, 64, 16, 5, 2
    rng = np.random.default_rng(30)
    L = b2.lib()
    pool = 80
    free = dev(torch, rng.permutation(pool), np.int32)
    state = dict(ctx=torch.zeros(batch, dtype=torch.int32, device="cuda"), mapped=torch.zeros(batch, dtype=torch.int32, device="cuda"),
                 count=dev(torch, [pool], np.int32))
    table = torch.full((batch, 12), -1, dtype=torch.int32, device="cuda")
    k, v = (torch.zeros(layers, pool, hkv, page, hd, device="cuda") for _ in range(2))
    freq = dev(torch, 1.0 / 10000.0 ** (np.arange(0, hd, 2) / hd), np.float32)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    hist = [[] for _ in range(batch)]    # per sequence: (position, k rows of the layers, v rows)
    for step in range(3):
        new = rng.integers(0, 30, batch)
        new[0] = 20
        rows = int(new.sum())
        start = np.concatenate([[0], np.cumsum(new)])
        trees = [make_tree(int(n), rng) for n in new]
        tree = dev(torch, np.array([m for t in trees for m in t[1]], np.uint64).view(np.int64))
        nd = dev(torch, new, np.int32)
        d = {x: torch.full((rows,), -1, dtype=torch.int32, device="cuda") for x in ("item", "pos", "slot")}
        rs = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
        mo, fo = torch.zeros_like(state["mapped"]), torch.zeros_like(state["count"])
        b2.check("plan", L.b2_kv_plan(b2.KvPlanArgs(
            batch=batch, max_rows=rows, page_tokens=page, pages_per_seq=12, pool_pages=pool, ctx_len=p(state["ctx"]), new_len=p(nd),
            tree=p(tree), mapped=p(state["mapped"]), free_pages=p(free), free_count=p(state["count"]), page_table=p(table),
            mapped_out=p(mo), free_out=p(fo), row_start=p(rs), row_item=p(d["item"]), row_pos=p(d["pos"]), row_slot=p(d["slot"]),
            err=p(err), pdl=1), None))
        state["mapped"], state["count"] = mo, fo
        ys = rng.normal(0, 1, (layers, rows, (h + 2 * hkv) * hd)).astype(np.float32)
        tokens, nxt = rng.integers(0, 3, rows), rng.integers(0, 3, rows)
        outs, keep = [], []
        for l in range(layers):
            y, q, o = dev(torch, ys[l]), torch.zeros(rows, h * hd, device="cuda"), torch.zeros(rows, h * hd, device="cuda")
            kv = b2.KVLayout(p(k[l]), p(v[l]), p(table), page, 12, hkv, hd)
            b2.check("append", L.b2_rows_append(b2.RowsAppendArgs(
                m=rows, y=p(y), y_stride=y.shape[1], q_rows=h * hd, q=p(q), q_stride=h * hd, rope_freq=p(freq), positions=p(d["pos"]),
                slots=p(d["slot"]), n_rows=rs.data_ptr() + 4 * batch, kv=kv, pool_pages=pool, err=p(err), pdl=1), None))
            a = b2.AttnRowsArgs(batch=batch, n_heads=h, n_kv_heads=hkv, head_dim=hd, max_rows=64, rows=rows, q=p(q), q_stride=h * hd,
                                kv=kv, pool_pages=pool, row_start=p(rs), ctx_len=p(state["ctx"]), tree=p(tree), max_ctx=12 * page,
                                ctx=p(o), ctx_stride=h * hd, err=p(err), pdl=1)
            sc = torch.empty(L.b2_attn_rows_scratch_bytes(a) + 16, dtype=torch.uint8, device="cuda")
            a.scratch, a.scratch_bytes = p(sc), sc.numel()
            b2.check("attn", L.b2_attn_rows(a, None))
            outs.append((q, o))
            keep += [y, sc]
        td = dev(torch, tokens, np.int32)
        kd = dev(torch, np.array([(0xC0000000 << 32) | (0xFFFFFFFF - int(t)) for t in nxt], np.uint64).view(np.int64))
        path = torch.zeros(batch, 64, dtype=torch.int32, device="cuda")
        cnt, follow, co = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(3))
        b2.check("accept", L.b2_tree_accept(b2.TreeAcceptArgs(
            batch=batch, max_rows=64, rows=rows, row_start=p(rs), tokens=p(td), tree=p(tree), argmax=p(kd), ctx_len=p(state["ctx"]),
            path=p(path), count=p(cnt), next=p(follow), ctx_out=p(co), err=p(err), pdl=1), None))
        kvs = (b2.KVLayout * layers)(*[b2.KVLayout(p(k[l]), p(v[l]), p(table), page, 12, hkv, hd) for l in range(layers)])
        b2.check("compact", L.b2_kv_compact(b2.KvCompactArgs(
            n_layers=layers, layers=kvs, pool_pages=pool, batch=batch, ctx_len=p(state["ctx"]), path=p(path), count=p(cnt), err=p(err),
            pdl=1), None))
        torch.cuda.synchronize()
        state["ctx"] = co
        assert int(err.item()) == 0
        # plain replay in float64
        def turn(x, pos):
            ang = (np.float32(pos) * freq.cpu().numpy()).astype(np.float64)
            r = x.astype(np.float64).copy()
            r[..., 0::2] = x[..., 0::2] * np.cos(ang) - x[..., 1::2] * np.sin(ang)
            r[..., 1::2] = x[..., 0::2] * np.sin(ang) + x[..., 1::2] * np.cos(ang)
            return r
        for b in range(batch):
            par, masks = trees[b]
            base = len(hist[b])
            nodes = []
            for i in range(int(new[b])):
                pos = base + bin(masks[i]).count("1") - 1
                yy = ys[:, start[b] + i].reshape(layers, h + 2 * hkv, hd)
                nodes.append((turn(yy[:, :h], pos), turn(yy[:, h:h + hkv], pos), yy[:, h + hkv:].astype(np.float64)))
            for i in range(int(new[b])):
                see = hist[b] + [nodes[j][1:] for j in range(int(new[b])) if masks[i] >> j & 1]
                K, V = np.stack([x[0] for x in see]), np.stack([x[1] for x in see])   # [t, layers, hkv, hd]
                for l in range(layers):
                    q = nodes[i][0][l].reshape(hkv, h // hkv, hd)
                    s = np.einsum("hgd,thd->hgt", q, K[:, l]) / np.sqrt(hd)
                    w = np.exp(s - s.max(-1, keepdims=True))
                    want = (np.einsum("hgt,thd->hgd", w, V[:, l]) / w.sum(-1)[..., None]).reshape(-1)
                    got = outs[l][1][start[b] + i].cpu().numpy()
                    # the keys and queries carry the append's 2^-21 too: twice the attention's bound
                    assert np.abs(got - want).max() <= 2 * ATTN_TOL * 5
            taken, _ = accept_reference(par if new[b] else [], tokens[start[b]:start[b + 1]], nxt[start[b]:start[b + 1]])
            assert list(path[b].cpu().numpy()[:len(taken)]) == taken and int(cnt[b]) == len(taken)
            hist[b] += [nodes[j][1:] for j in taken]
            tb = table[b].cpu().numpy()
            for at, (kk, vv) in enumerate(hist[b]):
                for l in range(layers):
                    assert np.abs(k[l, tb[at // page], :, at % page].cpu().numpy() - kk[l]).max() <= 2.0 ** -21 * 6
                    assert (v[l, tb[at // page], :, at % page].cpu().numpy() == vv[l].astype(np.float32)).all()
