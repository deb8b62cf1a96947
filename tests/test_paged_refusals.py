"""Refusals of the paged cache's calls, and where rows lie: argument checks that need no GPU (they come before the context's)."""
import ctypes as C

import numpy as np
import pytest

from conftest import load_pkg

pkg = load_pkg()
BAD = pkg.LV_ERR_BAD_ARGUMENTS
P = 1 << 20                      # a place that nothing looks at


def cache(**more):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, type=pkg.TYPE_I8, pages=10, page_rows=16, kv_heads=4, dim=64, table=P, table_ld=5, lens=P, starts=P, seqs=3)
    return pkg.PagedCache(**(a | more))


def attention(c=None, **more):
    a = dict(cache=c or cache(), q=P, q_type=pkg.TYPE_F32, q_ld=8 * 64, heads=8, tokens=6, max_new=3, max_len=80, scale=0.125, out=P, out_type=pkg.TYPE_BF16, out_ld=8 * 64)
    return pkg.PagedAttentionArgs(**(a | more))


def verification(**more):
    a = dict(target=P, target_ld=100, draft=P, draft_ld=100, vocab=100, drafted=P, starts=P, seqs=2, rows=7, accept=P, pick=P, tokens=P, accepted=P)
    return pkg.VerifyArgs(**(a | more))


def refused(rc, text):
    assert rc == BAD
    assert text in pkg.load_kernels().lv_last_error_string().decode(), pkg.load_kernels().lv_last_error_string()


BAD_CACHES = [(dict(k=None), "null"), (dict(table=None), "null"), (dict(lens=None), "null"), (dict(starts=None), "null"), (dict(type=pkg.TYPE_F32), "type"),
              (dict(type=pkg.TYPE_Q8_0), "type"), (dict(v_scale=None), "scales"), (dict(dim=0), "head size"), (dict(dim=72), "head size"), (dict(dim=272), "head size"),
              (dict(pages=0), "sizes"), (dict(page_rows=0), "sizes"), (dict(kv_heads=0), "sizes"), (dict(table_ld=0), "sizes"), (dict(seqs=0), "sizes"),
              (dict(seqs=65536), "sizes"), (dict(table_ld=1 << 30), "2^31"), (dict(v=P + 8), "aligned")]


@pytest.mark.parametrize("more,text", BAD_CACHES, ids=[f"{list(m)[0]}-{t[:8]}" for m, t in BAD_CACHES])
def test_caches_that_cannot_be(more, text):
    lib, c = pkg.load_kernels(), cache(**more)
    refused(lib.lv_paged_append(None, C.byref(c), P, P, pkg.TYPE_F32, 256, None, 0, 0, 3), text)
    refused(lib.lv_paged_read(None, C.byref(c), P, P, pkg.TYPE_F32, 0, 0, 0, 0, 3), text)
    a = attention(c)
    refused(lib.lv_paged_attention(None, C.byref(a), P, 1 << 30), text)
    assert lib.lv_paged_attention_scratch_bytes(None, C.byref(a)) == 0
    out = C.c_uint64()
    refused(lib.lv_paged_locate(C.byref(c), (C.c_uint32 * 5)(), 0, 0, C.byref(out)), text)


def test_calls_that_only_lack_a_context():
    lib, c, a, v = pkg.load_kernels(), cache(), attention(), verification()
    for rc in (lib.lv_paged_append(None, C.byref(c), P, P, pkg.TYPE_F32, 256, None, 0, 0, 3), lib.lv_paged_read(None, C.byref(c), P, P, pkg.TYPE_BF16, 0, 0, 64, 0, 3),
               lib.lv_paged_attention(None, C.byref(a), P, 1 << 30), lib.lv_probabilities(None, P, 10, P, 10, 10, 2, None), lib.lv_verify_drafts(None, C.byref(v))):
        refused(rc, "null context")


@pytest.mark.parametrize("args,text", [((None, P, 0, 256, None, 0, 0), "input"), ((P, P, 24, 256, None, 0, 0), "input"), ((P, P, 0, 255, None, 0, 0), "16-byte"), ((P, P, 0, 252, None, 0, 0), "16-byte"),
                                       ((P, P + 4, 0, 256, None, 0, 0), "16-byte"), ((P, P, 30, 260, None, 0, 0), "16-byte"), ((P, P, 0, 256, P, 64, 33), "angles"),
                                       ((P, P, 0, 256, P, 62, 32), "angles"), ((P, P, 0, 256, P + 4, 64, 32), "angles"), ((P, P, 0, 256, P, 65, 32), "angles")])
def test_appends_that_cannot_be(args, text):
    k, v, kind, ld, angles, angle_ld, pairs = args
    refused(pkg.load_kernels().lv_paged_append(None, C.byref(cache()), k, v, kind, ld, angles, angle_ld, pairs, 3), text)


@pytest.mark.parametrize("args,text", [((None, P, 0, 0, 0, 0), "output"), ((P, P, 259, 0, 0, 0), "output"), ((P, P, 0, 2, 0, 0), "16-byte"), ((P, P, 1, 0, 4, 0), "16-byte"), ((P, P, 30, 0, 0, 4), "16-byte"),
                                       ((P + 8, P, 0, 0, 0, 0), "16-byte")])
def test_reads_that_cannot_be(args, text):
    refused(pkg.load_kernels().lv_paged_read(None, C.byref(cache()), *args, 0, 3), text)


BAD_ATTENTION = [(dict(q=None), "null"), (dict(out=None), "null"), (dict(heads=0), "heads"), (dict(heads=6), "heads"), (dict(q_type=pkg.TYPE_I8), "type"), (dict(out_type=pkg.TYPE_E4M3), "type"),
                 (dict(q_ld=511), "strides"), (dict(out_ld=508), "strides"), (dict(q_ld=514), "16-byte"), (dict(out_ld=516), "16-byte"), (dict(q=P + 4), "16-byte"), (dict(out=P + 2), "16-byte"),
                 (dict(max_new=7), "bounds"), (dict(max_len=2), "bounds"), (dict(max_len=81), "bounds"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                 (dict(tokens=(1 << 31) - 1), "too many"), (dict(angles=P, angle_ld=64, angle_pairs=33), "angles")]


@pytest.mark.parametrize("more,text", BAD_ATTENTION, ids=[f"{i}-{t}" for i, (m, t) in enumerate(BAD_ATTENTION)])
def test_attentions_that_cannot_be(more, text):
    lib, a = pkg.load_kernels(), attention(**more)
    refused(lib.lv_paged_attention(None, C.byref(a), P, 1 << 30), text)
    assert lib.lv_paged_attention_scratch_bytes(None, C.byref(a)) == 0


def test_attention_wants_an_aligned_scratch():
    lib, a = pkg.load_kernels(), attention()
    refused(lib.lv_paged_attention(None, C.byref(a), None, 1 << 30), "scratch")
    refused(lib.lv_paged_attention(None, C.byref(a), P + 8, 1 << 30), "scratch")


@pytest.mark.parametrize("args", [(None, 10, P, 10, 10), (P, 10, None, 10, 10), (P, 9, P, 10, 10), (P, 10, P, 9, 10), (P, 0, P, 0, 0), (P, 1 << 25, P, 1 << 25, (1 << 24) + 1), (P, 11, P, 10, 10)])
def test_probabilities_that_cannot_be(args):
    assert pkg.load_kernels().lv_probabilities(None, *args, 2, None) == BAD
    assert b"null context" not in pkg.load_kernels().lv_last_error_string()


@pytest.mark.parametrize("more,text", [(dict(target=None), "null"), (dict(drafted=None), "null"), (dict(starts=None), "null"), (dict(accept=None), "null"), (dict(pick=None), "null"), (dict(tokens=None), "null"),
                                       (dict(accepted=None), "null"), (dict(vocab=0), "sizes"), (dict(target_ld=99), "sizes"), (dict(draft_ld=99), "sizes"), (dict(seqs=0), "rows"), (dict(rows=1 << 31), "rows")])
def test_verifications_that_cannot_be(more, text):
    a = verification(**more)
    refused(pkg.load_kernels().lv_verify_drafts(None, C.byref(a)), text)


def test_rows_lie_where_the_table_says():
    lib, out = pkg.load_kernels(), C.c_uint64()
    c = cache(pages=3_000_000, page_rows=20, kv_heads=8, dim=128, table_ld=4)
    row = (C.c_uint32 * 4)(5, 2_999_999, 0, 0xFFFFFFFF)
    for position, head in [(0, 0), (19, 7), (20, 3), (39, 7), (40, 0), (59, 1)]:
        assert lib.lv_paged_locate(C.byref(c), row, position, head, C.byref(out)) == pkg.LV_OK
        assert out.value == ((row[position // 20] * 8 + head) * 20 + position % 20) * 128
    assert np.uint64(2_999_999 * 8 * 20 * 128) > np.uint64(1 << 32)          # places beyond 32 bits
    refused(lib.lv_paged_locate(C.byref(c), row, 60, 0, C.byref(out)), "no page")          # a page that is not there
    refused(lib.lv_paged_locate(C.byref(c), row, 80, 0, C.byref(out)), "no such")          # behind the table
    refused(lib.lv_paged_locate(C.byref(c), row, 0, 8, C.byref(out)), "no such")


@pytest.mark.parametrize("page_rows", [1, 2, 3, 5, 7, 16, 20, 100, 127, 128, 129, 641, 65535, 65537, 1000003, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, (1 << 31) - 1])
def test_positions_are_divided_exactly(page_rows):
    """The multiplication that stands for the division by page_rows, at multiples of it, their neighbours and random positions."""
    lib, out = pkg.load_kernels(), C.c_uint64()
    slots = min(((1 << 31) - 1) // page_rows, 200000)
    c = cache(pages=slots, page_rows=page_rows, kv_heads=1, dim=16, table_ld=slots)
    table = np.arange(slots, dtype=np.uint32)
    row = table.ctypes.data_as(C.POINTER(C.c_uint32))
    most = slots * page_rows - 1
    rng = np.random.default_rng(page_rows)
    at = {0, most} | {int(m) * page_rows + e for m in rng.integers(0, slots, 300) for e in (-1, 0, 1)} | {int(p) for p in rng.integers(0, most + 1, 300)}
    for position in (p for p in at if 0 <= p <= most):
        assert lib.lv_paged_locate(C.byref(c), row, position, 0, C.byref(out)) == pkg.LV_OK
        assert out.value == position * 16
