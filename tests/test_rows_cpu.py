"""The row cache without a GPU: the header's symbols and struct layouts, the shapes, and every refusal of an argument (they come
before any device work, with a message)."""
import ctypes as C
import os
import re

import pytest

from redisearch_amd import rows as R
from redisearch_amd import vecsim as V

from . import rows_plain as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_symbols_are_bound_and_exported():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include/rsgpu_rows.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(RSGPU_\w+)\s*\(", src))
    assert names == set(R.ABI)
    lib = R.load()
    assert all(hasattr(lib, n) for n in names)


def test_header_compiles_as_c_and_cpp_and_structs_match(tmp_path):
    body = '#include <stdio.h>\n#include <stddef.h>\n#include "rsgpu_rows.h"\nint main(void){printf("%s", %s);return 0;}\n'
    fields = [("RSGPU_RowCache", R.RowCacheStruct), ("RSGPU_ScoreRules", R.ScoreRules)]
    wants, exprs = [], []
    for name, struct in fields:
        wants.append(C.sizeof(struct))
        exprs.append("sizeof(%s)" % name)
        for f, _ in struct._fields_:
            wants.append(getattr(struct, f).offset)
            exprs.append("offsetof(%s, %s)" % (name, f))
    text = body % (" ".join(["%zu"] * len(exprs)), ", ".join(exprs))
    for comp, ext in (("gcc -std=c99", "c"), ("g++ -std=c++11", "cpp")):
        f = tmp_path / ("t." + ext)
        f.write_text(text)
        exe = str(tmp_path / ("t_" + ext))
        assert os.system("%s -Wall -Werror -I%s/include %s -o %s" % (comp, ROOT, f, exe)) == 0
        assert [int(x) for x in os.popen(exe).read().split()] == wants


@pytest.mark.parametrize("vtype", [P.F32, P.F16, P.BF16])
@pytest.mark.parametrize("fmt", [R.NATIVE, R.INT8, R.E4M3, R.INT4])
@pytest.mark.parametrize("dim", [1, 31, 32, 33, 100, 128, 768, 65536])
def test_shapes(vtype, fmt, dim):
    for block in (0, 32, 64, 128):
        c = R.RowCache(vtype, dim, fmt, block)
        if fmt == R.NATIVE and block:
            assert c.row_bytes == 0 and c.row_scales == 0
        else:
            assert (c.row_bytes, c.row_scales) == (P.row_bytes(vtype, dim, fmt), P.row_scales(dim, fmt, block))


BUF = (C.c_char * 4096)()
AT = (C.addressof(BUF) + 63) // 64 * 64        # never read: a refused call launches nothing


def cache(**over):
    c = dict(vtype=P.F32, dim=96, fmt=R.INT8, block=32, capacity=8, codes=AT, scales=AT, device=0)
    c.update(over)
    return R.RowCache(c["vtype"], c["dim"], c["fmt"], c["block"], c["capacity"], c["codes"], c["scales"], c["device"])


BAD_CACHES = [dict(vtype=V.VecSimType_FLOAT64), dict(vtype=V.VecSimType_INT8), dict(vtype=99), dict(dim=0), dict(dim=65537), dict(fmt=4),
              dict(fmt=-1), dict(block=16), dict(block=96), dict(block=256), dict(fmt=R.NATIVE, block=32), dict(capacity=0),
              dict(capacity=1 << 49), dict(codes=None), dict(codes=AT + 8), dict(scales=None), dict(scales=AT + 2)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids="-".join)
def test_bad_caches_are_refused(bad):
    c = cache(**bad)
    with pytest.raises(RuntimeError, match="RSGPU_RowCache_Write: cache"):
        c.write(AT, 96, AT, 1)
    with pytest.raises(RuntimeError, match="RSGPU_RowCache_Read: cache"):
        c.read(AT, 1, AT, 96)
    with pytest.raises(RuntimeError, match="RSGPU_RowCache_PartitionScores: cache"):
        c.partition_scores(AT, 96, 1, AT, 1, AT, 1, 16, AT, R.PRODUCT, AT, 16)


@pytest.mark.parametrize("bad", [dict(rows=None), dict(slots=None), dict(stride=95), dict(stride=1 << 62), dict(rows=AT + 2),
                                 dict(slots=AT + 4), dict(n=1 << 31)], ids="-".join)
def test_bad_writes_and_reads_are_refused(bad):
    a = dict(rows=AT, stride=96, slots=AT, n=2)
    a.update(bad)
    with pytest.raises(RuntimeError, match="RSGPU_RowCache_Write: "):
        cache().write(a["rows"], a["stride"], a["slots"], a["n"])
    with pytest.raises(RuntimeError, match="RSGPU_RowCache_Read: "):
        cache().read(a["slots"], a["n"], a["rows"], a["stride"])


SCORES = dict(queries=AT, stride=96, n_queries=2, query_offsets=AT, n_partitions=2, pages=AT, max_pages=3, page_rows=16, row_counts=AT,
              form=R.PRODUCT, scores=AT, ld=48)


@pytest.mark.parametrize("bad", [dict(queries=None), dict(query_offsets=None), dict(pages=None), dict(row_counts=None), dict(scores=None),
                                 dict(stride=95), dict(stride=1 << 62), dict(n_queries=1 << 31), dict(n_partitions=1 << 31),
                                 dict(max_pages=1 << 31), dict(page_rows=0), dict(page_rows=1 << 31), dict(form=2), dict(form=-1),
                                 dict(ld=1 << 62), dict(queries=AT + 2), dict(query_offsets=AT + 1), dict(pages=AT + 2),
                                 dict(row_counts=AT + 3), dict(scores=AT + 2)], ids="-".join)
def test_bad_scores_are_refused(bad):
    with pytest.raises(RuntimeError, match="RSGPU_RowCache_PartitionScores: "):
        cache().partition_scores(**{**SCORES, **bad})


RULES = dict(form=R.PRODUCT, device=0, mask=AT, mask_words=4, n_masks=2, bias_offsets=AT, bias_ids=AT, bias_values=AT, n_bias=3,
             seen_offsets=AT, seen_ids=AT, n_seen=3, repetition=AT, frequency=AT, presence=AT)


@pytest.mark.parametrize("bad", [dict(form=2), dict(mask_words=3), dict(n_masks=1), dict(bias_ids=None), dict(bias_values=None),
                                 dict(seen_ids=None), dict(n_bias=1 << 31), dict(n_seen=1 << 31), dict(mask=AT + 1),
                                 dict(mask_rows=AT + 1), dict(seen_offsets=AT + 2), dict(repetition=AT + 2)], ids="-".join)
def test_bad_rules_are_refused(bad):
    with pytest.raises(RuntimeError, match="RSGPU_AdjustScores: "):
        R.adjust_scores(R.score_rules(**{**RULES, **bad}), AT, AT, 2, 128, 128)


@pytest.mark.parametrize("bad", [dict(scores_in=None), dict(scores_out=None), dict(scores_in=AT + 1), dict(ld=127), dict(n_queries=1 << 31),
                                 dict(n_columns=1 << 31, ld=1 << 31), dict(ld=1 << 62), dict(counts=AT + 2)], ids="-".join)
def test_bad_adjustments_are_refused(bad):
    a = {**dict(scores_in=AT, scores_out=AT, n_queries=2, n_columns=128, ld=128), **bad}
    rules = R.score_rules(device=0)
    with pytest.raises(RuntimeError, match="RSGPU_AdjustScores: "):
        R.adjust_scores(rules, **a)


def test_no_structs_are_refused():
    lib = R.load()
    assert lib.RSGPU_RowCache_Write(None, AT, 96, AT, 1, None) == -1
    assert lib.RSGPU_RowCache_Read(None, AT, 1, AT, 96, None) == -1
    assert lib.RSGPU_AdjustScores(None, AT, AT, 1, 1, 1, None, None) == -1
    assert lib.RSGPU_FlatIndex_CacheRows(None, 0, 1, cache().ref, AT, None) == -1
    assert lib.RSGPU_FlatIndex_AddCachedRows(None, cache().ref, AT, 1, 1, None) == -1
    assert lib.RSGPU_RowCache_RowBytes(None) == 0 and lib.RSGPU_RowCache_RowScales(None) == 0


def test_nothing_to_do_is_no_error():
    cache().write(None, 0, None, 0)
    cache().read(None, 0, None, 0)
    for none in ("n_queries", "n_partitions", "max_pages", "ld"):
        cache().partition_scores(**{**SCORES, none: 0})
    R.adjust_scores(R.score_rules(device=0), None, None, 0, 128, 128)
    R.adjust_scores(R.score_rules(device=0), None, None, 2, 0, 0)


def test_plain_e4m3_rounds_to_nearest_even():
    table = P.e4m3_values()[:127]
    assert (P.e4m3_code(table) == range(127)).all()
    mid = (table[:-1] + table[1:]) / 2
    assert (P.e4m3_code(mid) % 2 == 0).all()
