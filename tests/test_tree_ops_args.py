"""Arguments that the operators of several new rows per sequence refuse before
any device work (no GPU needed): every wrong call returns its code, and the
struct it was given stays as it was."""
import ctypes as C

import numpy as np
import pytest

_KEEP = np.zeros(4096 + 64, np.uint8)
P = (_KEEP.ctypes.data + 63) // 64 * 64   # aligned stand-in for device memory: never dereferenced


def kv(b2, **over):
    a = b2.KVLayout(P, P, P, 16, 4, 2, 64)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def attn(b2):
    return b2.AttnRowsArgs(batch=2, n_heads=4, n_kv_heads=2, head_dim=64, max_rows=4, rows=8, q=P, q_stride=256, kv=kv(b2),
                           row_start=P, ctx_len=P, tree=P, max_ctx=64, ctx=P, ctx_stride=256, scratch=P, scratch_bytes=1 << 30)


def plan(b2):
    return b2.KvPlanArgs(batch=2, max_rows=8, page_tokens=16, pages_per_seq=4, pool_pages=8, ctx_len=P, new_len=P, tree=P, mapped=P,
                         free_pages=P, free_count=P, page_table=P, mapped_out=P + 64, free_out=P + 64, row_start=P, row_item=P,
                         row_pos=P, row_slot=P)


def append(b2):
    return b2.RowsAppendArgs(m=4, y=P, y_stride=512, q_rows=256, q=P, q_stride=256, rope_freq=P, positions=P, slots=P, kv=kv(b2),
                             pool_pages=8)


def accept(b2):
    return b2.TreeAcceptArgs(batch=2, max_rows=8, rows=8, row_start=P, tokens=P, tree=P, argmax=P, ctx_len=P, path=P, count=P, next=P,
                             ctx_out=P)


def compact(b2, layers=2, **over):
    k = (b2.KVLayout * layers)(*[kv(b2) for _ in range(layers)])
    for name, v in over.items():
        setattr(k[layers - 1], name, v)
    return b2.KvCompactArgs(n_layers=layers, layers=k, batch=2, ctx_len=P, path=P, count=P)


CASES = {
    "b2_attn_rows": (attn, [
        dict(batch=0), dict(batch=65536), dict(n_heads=0), dict(n_kv_heads=0), dict(n_heads=5), dict(head_dim=0), dict(head_dim=144),
        dict(head_dim=40), dict(head_dim=128), dict(max_rows=0), dict(rows=0), dict(q=None), dict(q=P + 4), dict(q_stride=252),
        dict(q_stride=258), dict(ctx=None), dict(ctx=P + 8), dict(ctx_stride=252), dict(ctx_stride=257), dict(row_start=None),
        dict(ctx_len=None), dict(max_ctx=0), dict(max_ctx=65), dict(max_rows=0x80000000), dict(rows=0x80000000)]),
    "b2_kv_plan": (plan, [
        dict(batch=0), dict(max_rows=0), dict(page_tokens=0), dict(pages_per_seq=0), dict(pool_pages=0), dict(ctx_len=None),
        dict(new_len=None), dict(mapped=None), dict(free_pages=None), dict(free_count=None), dict(page_table=None),
        dict(mapped_out=None), dict(free_out=None), dict(row_start=None), dict(row_item=None), dict(row_pos=None),
        dict(row_slot=None), dict(mapped_out=P), dict(free_out=P), dict(max_rows=0x80000000), dict(pages_per_seq=1 << 28),
        dict(pool_pages=1 << 28)]),
    "b2_rows_append": (append, [
        dict(m=0), dict(y=None), dict(y=P + 4), dict(y_stride=508), dict(y_stride=514), dict(q_rows=0), dict(q_rows=250), dict(q=None),
        dict(q=P + 4), dict(q_stride=252), dict(q_stride=257), dict(positions=None), dict(slots=None), dict(pool_pages=0),
        dict(pool_pages=1 << 28), dict(m=0x80000000)]),
    "b2_tree_accept": (accept, [
        dict(batch=0), dict(max_rows=0), dict(max_rows=65), dict(row_start=None), dict(tokens=None), dict(argmax=None),
        dict(ctx_len=None), dict(path=None), dict(count=None), dict(next=None), dict(ctx_out=None), dict(rows=0x80000000)]),
    "b2_kv_compact": (compact, [
        dict(n_layers=0), dict(batch=0), dict(batch=65536), dict(ctx_len=None), dict(path=None), dict(count=None)]),
}


@pytest.mark.parametrize("fn,change", [(f, c) for f, (_, cs) in CASES.items() for c in cs], ids=str)
def test_refused(b2, fn, change):
    a = CASES[fn][0](b2)
    for k, v in change.items():
        setattr(a, k, v)
    before = bytes(a)
    assert getattr(b2.lib(), fn)(a, None) == -1
    assert bytes(a) == before


@pytest.mark.parametrize("fn", list(CASES))
def test_null_refused(b2, fn):
    assert getattr(b2.lib(), fn)(None, None) == -1


@pytest.mark.parametrize("change", [dict(k_pool=None), dict(v_pool=None), dict(page_table=None), dict(page_tokens=0), dict(head_dim=48),
                                    dict(n_kv_heads=4), dict(k_pool=P + 4), dict(pages_per_seq=0), dict(pages_per_seq=1 << 28)])
def test_attn_layout_refused(b2, change):
    a = attn(b2)
    a.kv = kv(b2, **change)
    assert b2.lib().b2_attn_rows(a, None) == -1
    assert b2.lib().b2_attn_rows_scratch_bytes(a) == 0


@pytest.mark.parametrize("change", [dict(k_pool=None), dict(v_pool=P + 4), dict(page_table=None), dict(page_tokens=8),
                                    dict(pages_per_seq=5), dict(n_kv_heads=3), dict(head_dim=32), dict(pages_per_seq=0)])
def test_compact_layers_refused(b2, change):
    assert b2.lib().b2_kv_compact(compact(b2, **change), None) == -1


def test_batches_past_the_plan_unsupported(b2):
    a = plan(b2)
    a.batch = 4097
    assert b2.lib().b2_kv_plan(a, None) == -9


def test_python_structs_match_the_header(b2, tmp_path):
    """Sizes and field offsets of the ctypes mirrors against the C compiler's."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"b2_kv_plan_args": b2.KvPlanArgs, "b2_rows_append_args": b2.RowsAppendArgs, "b2_attn_rows_args": b2.AttnRowsArgs,
             "b2_tree_accept_args": b2.TreeAcceptArgs, "b2_kv_compact_args": b2.KvCompactArgs}
    src = ['#include "b2_kernels.h"', "#include <stdio.h>", "int main(void) {"]
    for n, t in names.items():
        src.append(f'printf("%zu\\n", sizeof({n}));')
        src += [f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in t._fields_]
    (tmp_path / "s.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    want = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    got = []
    for t in names.values():
        got += [C.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want
