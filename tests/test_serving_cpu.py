"""CPU checks of the serving operators (include/ft_serving.h): refusals before any CUDA call, rotary frequencies, tree
masks and the page pool, which are host functions."""
import ctypes
import math
import os
import random
import re
import subprocess
import threading
import time
import types
import unittest.mock

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "ft_serving.h")


@pytest.fixture(scope="module")
def ftg(lib_path):
    import ft_gemm_b200
    return ft_gemm_b200


@pytest.fixture(scope="module")
def sv(ftg):
    from ft_gemm_b200 import serving
    serving._lib()
    return serving


def test_library_exports_every_declared_symbol(lib_path):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(ft_[a-z0-9_]+)\s*\(", text))
    assert {"ft_rotary_run", "ft_kv_cache_append", "ft_prompt_attention_run", "ft_tree_attention_run"} <= names
    out = subprocess.run(["nm", "-D", "--defined-only", lib_path], capture_output=True, text=True, check=True).stdout
    for name in names:
        assert re.search(rf"\bT {name}\b", out), name


def test_header_is_c_and_struct_sizes_match(tmp_path, sv):
    src = tmp_path / "s.c"
    names = ["ft_rows", "ft_rotary_options", "ft_kv_cache", "ft_prompt_attention_args", "ft_tree_attention_args"]
    src.write_text('#include <stdio.h>\n#include "ft_serving.h"\nint main(void){printf("' + "%zu " * len(names) + '\\n", '
                   + ", ".join(f"sizeof({n})" for n in names) + "); return 0;}\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    sizes = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(t) for t in (sv.FtRows, sv.FtRotaryOptions, sv.FtKvCache, sv.FtPromptAttentionArgs, sv.FtTreeAttentionArgs)]


def _frequencies(sv, **fields):
    o = sv.FtRotaryOptions()
    sv._lib().ft_rotary_options_default(ctypes.byref(o), fields.pop("head_dim", 128))
    for name, value in fields.items():
        setattr(o, name, value)
    out = (ctypes.c_double * 128)()
    return sv._lib().ft_rotary_frequencies(ctypes.byref(o), out), list(out[:max(0, min(256, o.rotary_dim)) // 2])


@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
def test_rotary_frequencies(sv, ftg, scaling):
    code, got = _frequencies(sv, rotary_dim=96, scaling=scaling, base=500000.0, factor=8.0, original_length=8192.0)
    assert code == ftg.FT_OK
    for i, g in enumerate(got):
        f = math.exp(-2 * i / 96 * math.log(500000.0 * (8 ** (96 / 94) if scaling == 2 else 1)))
        if scaling == 1:
            f /= 8
        if scaling == 3:
            turns = 8192 * f / (2 * math.pi)
            keep = 1.0 if turns >= 4 else 0.0 if turns <= 1 else (turns - 1) / 3
            f = f * keep + f / 8 * (1 - keep)
        assert g == pytest.approx(f, rel=1e-13)


def test_rotary_refusals(sv, ftg):
    for bad in (dict(rotary_dim=0), dict(rotary_dim=24), dict(rotary_dim=144), dict(head_dim=72), dict(head_dim=512), dict(base=0.0),
                dict(base=math.nan), dict(factor=0.0), dict(factor=-1.0), dict(magnitude=math.inf), dict(scaling=4), dict(scaling=-1),
                dict(scaling=3), dict(scaling=3, original_length=8192.0, low=4.0, high=4.0)):
        assert _frequencies(sv, **bad)[0] == ftg.FT_ERR_INVALID, bad
    lib, rows = sv._lib(), sv.FtRows(0x1000, 128, 128, 1)
    assert lib.ft_rotary_run(None, rows, rows, None, None, None, 1, 1, 0, None) == ftg.FT_ERR_INVALID
    assert lib.ft_rotary_prepare(None, None, None) == ftg.FT_ERR_INVALID
    assert lib.ft_rotary_destroy(None) == ftg.FT_OK


def _cache(sv, **fields):
    c = sv.FtKvCache(0x10000, 0x20000, 2 * 4 * 16 * 2 * 64, 16 * 2 * 64, 2 * 64, 64, 2, 4, 16, 2, 64, 1)
    for name, value in fields.items():
        setattr(c, name, value)
    return c


def test_cache_refusals(sv, ftg):
    lib = sv._lib()
    assert lib.ft_kv_cache_copy_pages(_cache(sv), None, None, 0, None) == ftg.FT_OK
    for bad in (dict(k=None), dict(v=None), dict(k=0x10008), dict(dtype=0), dict(layers=0), dict(pages=0), dict(kv_heads=0), dict(head_dim=96),
                dict(page_size=24), dict(page_size=4), dict(page_size=512), dict(token_stride=64), dict(head_stride=128), dict(page_stride=2047),
                dict(page_stride=1024), dict(layer_stride=8193)):
        assert lib.ft_kv_cache_copy_pages(_cache(sv, **bad), None, None, 0, None) == ftg.FT_ERR_INVALID, bad
    assert lib.ft_kv_cache_copy_pages(None, None, None, 0, None) == ftg.FT_ERR_INVALID
    assert lib.ft_kv_cache_copy_pages(_cache(sv), None, None, 1, None) == ftg.FT_ERR_INVALID
    assert lib.ft_kv_cache_copy_pages(_cache(sv), 0x1000, 0x1000, -1, None) == ftg.FT_ERR_INVALID
    # by head: a page [kv_heads][page_size][head_dim]
    assert lib.ft_kv_cache_copy_pages(_cache(sv, token_stride=64, head_stride=16 * 64), None, None, 0, None) == ftg.FT_OK
    good = sv.FtRows(0x1000, 128, 64, 2)
    for k, v, slots, layer, rotary, q in ((None, good, 0x1000, 0, None, None), (good, None, 0x1000, 0, None, None), (good, good, None, 0, None, None),
                                          (good, good, 0x1000, 2, None, None), (good, good, 0x1000, -1, None, None),
                                          (good, good, 0x1000, 0, None, good), (sv.FtRows(0x1000, 128, 64, 3), good, 0x1000, 0, None, None),
                                          (sv.FtRows(0x1004, 128, 64, 2), good, 0x1000, 0, None, None),
                                          (sv.FtRows(0x1000, 130, 64, 2), good, 0x1000, 0, None, None)):
        assert lib.ft_kv_cache_append(_cache(sv), layer, k, v, slots, 1, rotary, None, q, q, None) == ftg.FT_ERR_INVALID
    x = 0x1000
    assert lib.ft_kv_cache_accept(_cache(sv), x, 4, 4, x, x, x, x, 1, x, None) == ftg.FT_ERR_INVALID and b"lengths array" in lib.ft_gemm_last_error()
    assert lib.ft_kv_cache_accept(_cache(sv), x, 4, 3, x, x, x, x, 1, x + 64, None) == ftg.FT_ERR_INVALID
    assert lib.ft_kv_cache_accept(_cache(sv), None, 4, 4, x, x, x, x, 1, x + 64, None) == ftg.FT_ERR_INVALID


def test_attention_refusals(sv, ftg):
    lib = sv._lib()
    size = 1 << 40  # of the workspace, said only

    def prompt(workspace=0x100000, status=0x1000, **fields):
        r = lambda heads: sv.FtRows(0x10000, heads * 128, 128, heads)  # noqa: E731
        a = sv.FtPromptAttentionArgs(r(8), r(2), r(2), r(8), None, 0x1000, None, 1, 16, 16, 128, 1, 1, 0.0)
        for name, value in fields.items():
            setattr(a, name, value)
        return lib.ft_prompt_attention_run(a, workspace, size, status, None)

    rows = sv.FtRows
    for bad in (dict(workspace=None), dict(workspace=0x100008), dict(status=None), dict(dtype=0), dict(dtype=3), dict(head_dim=96), dict(head_dim=256),
                dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(batch=-1), dict(query_tokens=-1), dict(q_offsets=None),
                dict(q=rows(0x10000, 1024, 128, 7)), dict(q=rows(0x10000, 1024, 128, 0)), dict(q=rows(0x10000, 65 * 512, 128, 258)),
                dict(q=rows(None, 1024, 128, 8)), dict(q=rows(0x10002, 1024, 128, 8)), dict(k=rows(0x10000, 257, 128, 2)),
                dict(v=rows(0x10000, 256, 128, 3)), dict(out=rows(0x10000, 1024, 128, 4)), dict(out=rows(0x10000, 1024, 4, 8))):
        assert prompt(**bad) == ftg.FT_ERR_INVALID, bad
    assert lib.ft_prompt_attention_run(None, 0x100000, size, 0x1000, None) == ftg.FT_ERR_INVALID
    assert prompt(batch=0) == ftg.FT_OK and prompt(query_tokens=0) == ftg.FT_OK

    def tree(cache=None, workspace=0x100000, bytes_=size, status=0x1000, **fields):
        r = sv.FtRows(0x10000, 4 * 64, 64, 4)
        a = sv.FtTreeAttentionArgs(r, r, None, 0x1000, 0x1000, 0x1000, None, 0, 0, 1, 4, 4, 4, 0, 0.0)
        for name, value in fields.items():
            setattr(a, name, value)
        return lib.ft_tree_attention_run(cache or _cache(sv), a, workspace, bytes_, status, None)

    for bad in (dict(cache=_cache(sv, page_size=12)), dict(workspace=None), dict(bytes_=0), dict(status=None), dict(layer=2), dict(layer=-1),
                dict(table_pages=0), dict(table_stride=3), dict(table_pages=1 << 28, table_stride=1 << 28), dict(mask=0x1000), dict(mask=0x1000, mask_words=2, mask_stride=1),
                dict(batch=-1), dict(q_offsets=None), dict(page_table=None), dict(lengths=None), dict(scale=-0.5),
                dict(q=rows(0x10000, 192, 64, 3)), dict(out=rows(0x10008, 256, 64, 4))):
        assert tree(**bad) == ftg.FT_ERR_INVALID, bad
    assert tree(batch=0) == ftg.FT_OK


def test_python_refuses_what_is_not_a_cuda_cache(ftg):
    torch = pytest.importorskip("torch")
    k = torch.empty((1, 2, 16, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ftg.PagedCache(k, k.clone())
    with pytest.raises(ValueError, match="scaling"):
        ftg.Rotary(128, scaling="by parts")
    with pytest.raises(ftg.FtGemmError, match="multiples of 16"):
        ftg.Rotary(128, rotary_dim=40)
    with pytest.raises(ValueError, match="element type"):
        ftg.PromptAttention(8, 2, 128, dtype=torch.float32)


SCHEDULE = r"""
#include <cstdio>
#include <cstdlib>
#include "serving_schedule.h"
using namespace ftg;
// the units of a row tile, from the definition
static int units(int n, int keys, int full, int per_item, int cost, bool chain, int r) {
  const int end = (r + 1) * per_item < n ? (r + 1) * per_item : n;
  int seen = chain && keys == full ? full - n + end : keys;  // keys that the tile's last row sees
  if (seen < 1) seen = 1;
  return (seen + 127) / 128 + cost;
}
int main() {
  srand(7);
  for (int i = 0; i < 30000; ++i) {
    const int per_item = 1 + rand() % 256, n = rand() % (i % 3 ? 300 : 3000), full = i % 5 ? rand() % 3000 : rand() % 20;
    const int keys = i % 7 == 0 && full ? rand() % full : full, cost = rand() % 4;
    const bool chain = rand() % 3 != 0;
    const SequenceTiles s = SequenceTiles::make(n, keys, full, per_item, cost, chain);
    if (s.row_tiles != (n + per_item - 1) / per_item) return printf("row tiles\n"), 1;
    int sum = 0;
    for (int r = 0; r < s.row_tiles; ++r) {
      if (s.units_before(r) != sum || s.units_of(r) != units(n, keys, full, per_item, cost, chain, r)) return printf("row tile %d of case %d\n", r, i), 1;
      sum += s.units_of(r);
    }
    if (s.units_per_head() != sum) return printf("case %d\n", i), 1;
  }
  // the largest numbers: 2^30 keys
  const SequenceTiles s = SequenceTiles::make(1, 1 << 30, 1 << 30, 32, 2, true);
  return s.units_of(0) == (1 << 23) + 2 && s.units_per_head() == s.units_of(0) ? 0 : 1;
}
"""


def test_shares_of_work_are_numbered_without_gaps(tmp_path):
    """The closed forms that every CTA finds its share with, against counting (host build of the device code)."""
    (tmp_path / "s.cpp").write_text(SCHEDULE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "ft_gemm_b200", "csrc"),
                    str(tmp_path / "s.cpp"), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


def test_tree_mask(ftg):
    pytest.importorskip("torch")
    rng = random.Random(3)
    for nodes, words in ((0, 0), (1, None), (33, None), (70, 4)):
        parents = [rng.randint(-1, i - 1) for i in range(nodes)]
        got = ftg.tree_mask(parents, words)
        for i in range(nodes):
            want, j = set(), i
            while j >= 0:
                want.add(j)
                j = parents[j]
            row = [int(w) & 0xFFFFFFFF for w in got[i]]
            assert {j for j in range(32 * len(row)) if row[j // 32] >> (j % 32) & 1} == want
    with pytest.raises(ftg.FtGemmError, match="before their children"):
        ftg.tree_mask([-1, 1])
    with pytest.raises(ftg.FtGemmError, match="bits"):
        ftg.tree_mask([-1] * 33, 1)


def test_page_pool_against_a_model(ftg):
    """Random calls; the contents of every page are modelled on the side, and pages are copied as the pool says."""
    pytest.importorskip("torch")
    rng = random.Random(11)
    for size, pages in ((1, 30), (4, 24), (16, 9)):
        pool, store, want, token = ftg.PagePool(pages, size), [[None] * size for _ in range(pages)], {}, 0
        for _ in range(600):
            act = rng.choice(["new", "extend", "extend", "extend", "fork", "free", "truncate", "compact"])
            some = rng.choice(list(want)) if want else None
            if act == "new" and len(want) < 8:
                want[pool.new_sequence()] = []
            elif some is None:
                continue
            elif act == "extend":
                count, free = rng.randint(0, 2 * size + 1), pool.free_pages()
                before = pool.page_list(some)
                try:
                    pairs = pool.extend([some], [count])
                except ftg.FtGemmError:
                    assert pool.free_pages() == free and pool.page_list(some) == before and pool.length(some) == len(want[some])
                    continue
                for a, b in pairs:
                    store[b] = list(store[a])
                first = len(want[some])
                for slot in pool.slots(some, first, count):
                    store[slot // size][slot % size] = token
                    want[some].append(token)
                    token += 1
            elif act == "fork" and len(want) < 8:
                want[pool.fork(some)] = list(want[some])
            elif act == "free":
                pool.free(some)
                del want[some]
            elif act == "truncate":
                length = rng.randint(0, len(want[some]))
                pool.truncate(some, length)
                del want[some][length:]
            elif act == "compact":
                pairs = pool.compact()
                assert not {a for a, _ in pairs} & {b for _, b in pairs}
                for a, b in pairs:
                    store[b] = list(store[a])
            used = {p for s in want for p in pool.page_list(s)}
            assert pool.free_pages() == pages - len(used)
            if act == "compact":
                assert used == set(range(len(used)))
            for s, tokens in want.items():
                assert pool.length(s) == len(tokens)
                assert [store[x // size][x % size] for x in pool.slots(s, 0, len(tokens))] == tokens
        for s in list(want):
            pool.free(s)
        assert pool.free_pages() == pages
        with pytest.raises(ftg.FtGemmError, match="no sequence"):
            pool.free(0)
        with pytest.raises(ftg.FtGemmError):
            pool.fork(-1)
        pool.close()


def test_page_pool_refusals(ftg, sv):
    pytest.importorskip("torch")
    lib, handle = sv._lib(), ctypes.c_void_p()
    assert lib.ft_page_pool_create(ctypes.byref(handle), 0, 16) == ftg.FT_ERR_INVALID
    assert lib.ft_page_pool_create(ctypes.byref(handle), 4, 0) == ftg.FT_ERR_INVALID
    assert lib.ft_page_pool_create(None, 4, 16) == ftg.FT_ERR_INVALID
    assert lib.ft_page_pool_free_pages(None) == ftg.FT_ERR_INVALID
    assert lib.ft_page_pool_destroy(None) == ftg.FT_OK
    pool = ftg.PagePool(4, 16)
    s = pool.new_sequence()
    with pytest.raises(ftg.FtGemmError, match="free pages"):
        pool.extend([s], [65])
    with pytest.raises(ftg.FtGemmError):
        pool.extend([s], [-1])
    with pytest.raises(ftg.FtGemmError):
        pool.extend([s], [2 ** 31 - 1])
    with pytest.raises(ftg.FtGemmError):
        pool.truncate(s, 1)
    with pytest.raises(ValueError):
        pool.slots(s, 0, 1)
    with pytest.raises(ValueError):
        pool.extend([s], [1, 2])


def test_sizes_that_a_launch_cannot_count_are_refused(sv, ftg):
    lib = sv._lib()
    # key heads beyond 8192: a page's elements would pass 31 bits
    many = _cache(sv, kv_heads=8193, page_size=256, token_stride=8193 * 64, page_stride=256 * 8193 * 64)
    assert lib.ft_kv_cache_copy_pages(many, None, None, 0, None) == ftg.FT_ERR_INVALID
    # a page of 256 x 8192 x 128 elements is 32768 pieces of 16 KiB: 2^16 of them pass 2^31 - 1 blocks
    large = _cache(sv, kv_heads=8192, page_size=256, head_dim=128, token_stride=8192 * 128, head_stride=128, page_stride=256 * 8192 * 128,
                   layer_stride=1 << 40)
    assert lib.ft_kv_cache_copy_pages(large, None, None, 0, None) == ftg.FT_OK
    assert lib.ft_kv_cache_copy_pages(large, 0x1000, 0x2000, 1 << 16, None) == ftg.FT_ERR_INVALID
    assert b"at most 65535" in lib.ft_gemm_last_error()
    # rotary positions: 2^30 tokens, 2^20 heads
    rows, rotary = sv.FtRows(0x1000, 64, 64, 1), 0x1000
    wide = sv.FtRows(0x1000, 64, 0, (1 << 20) + 1)
    assert lib.ft_rotary_run(rotary, rows, rows, None, None, 0x1000, (1 << 30) + 1, 1, 0, None) == ftg.FT_ERR_INVALID
    assert lib.ft_rotary_run(rotary, wide, wide, None, None, 0x1000, 1, 1, 0, None) == ftg.FT_ERR_INVALID
    assert lib.ft_rotary_run(rotary, rows, rows, wide, wide, 0x1000, 1, 1, 0, None) == ftg.FT_ERR_INVALID
    good = sv.FtRows(0x1000, 128, 64, 2)
    assert lib.ft_kv_cache_append(_cache(sv), 0, good, good, 0x1000, (1 << 30) + 1, None, None, None, None, None) == ftg.FT_ERR_INVALID
    # attention: 2^27 keys, 2^30 queries
    r = lambda heads: sv.FtRows(0x10000, heads * 128, 128, heads)  # noqa: E731
    for queries, keys in ((16, (1 << 27) + 1), ((1 << 30) + 1, 16)):
        a = sv.FtPromptAttentionArgs(r(8), r(2), r(2), r(8), None, 0x1000, 0x1000, 1, queries, keys, 128, 1, 1, 0.0)
        assert lib.ft_prompt_attention_run(a, 0x100000, 1 << 40, 0x1000, None) == ftg.FT_ERR_INVALID
        assert b"2^27 keys" in lib.ft_gemm_last_error()
    x = sv.FtRows(0x10000, 4 * 64, 64, 4)
    for pages in ((1 << 27) // 16 + 1, 2 ** 31 - 1):
        a = sv.FtTreeAttentionArgs(x, x, None, 0x1000, 0x1000, 0x1000, None, 0, 0, 1, 4, pages, pages, 0, 0.0)
        assert lib.ft_tree_attention_run(_cache(sv), a, 0x100000, 1 << 40, 0x1000, None) == ftg.FT_ERR_INVALID
        assert b"2^27 tokens" in lib.ft_gemm_last_error()
    # pages that do not begin on a group of 8 tokens
    a = sv.FtTreeAttentionArgs(x, x, None, 0x1000, 0x1000, 0x1000, None, 0, 0, 1, 4, 4, 4, 0, 0.0)
    assert lib.ft_tree_attention_run(_cache(sv, page_stride=16 * 2 * 64 + 64), a, 0x100000, 1 << 40, 0x1000, None) == ftg.FT_ERR_INVALID
    assert b"page stride" in lib.ft_gemm_last_error()


class _Handle(ctypes.Structure):
    """A rotary handle as the library lays it out, for calls that are refused before they look at the frequencies."""


def _handle(sv, head_dim):
    if not hasattr(_Handle, "_fields_"):
        _Handle._fields_ = [("options", sv.FtRotaryOptions), ("turns", ctypes.c_void_p)]
    h = _Handle()
    sv._lib().ft_rotary_options_default(ctypes.byref(h.options), head_dim)
    return h


def _share(strides, counts, block):
    """Do two blocks at i * strides[0] + j * strides[1] share an element?"""
    at = sorted(i * strides[0] + j * strides[1] for i in range(counts[0]) for j in range(counts[1]))
    return any(b - a < block for a, b in zip(at, at[1:]))


def test_outputs_whose_rows_share_memory_are_refused(sv, ftg):
    """Expanded outputs, and all others in which two rows meet, from the definition; what is refused never reaches a device."""
    lib, rng, refused = sv._lib(), random.Random(5), 0
    shapes = [((0, 64), (4, 2)), ((64, 64), (4, 2)), ((128, 0), (4, 2)), ((64, 128), (4, 2)), ((32, 256), (4, 2))]
    for _ in range(3000):
        shapes.append(((8 * rng.randint(0, 40), 8 * rng.randint(0, 40)), (rng.randint(1, 9), rng.randint(1, 9))))
    h = _handle(sv, 64)
    for (token, head), (tokens, heads) in shapes:
        if not _share((token, head), (tokens, heads), 64):
            continue
        refused += 1
        fine, bad = sv.FtRows(0x100000, heads * 64, 64, heads), sv.FtRows(0x200000, token, head, heads)
        for q_out, k, k_out in ((bad, None, None), (fine, fine, bad)):
            q = sv.FtRows(0x300000, heads * 64, 64, heads)
            assert lib.ft_rotary_run(ctypes.byref(h), q, q_out, k, k_out, 0x1000, tokens, 1, 0, None) == ftg.FT_ERR_INVALID
            assert b"share memory" in lib.ft_gemm_last_error()
        kv = sv.FtRows(0x100000, 128, 64, 2)
        assert lib.ft_kv_cache_append(_cache(sv), 0, kv, kv, 0x1000, tokens, ctypes.byref(h), 0x1000, fine, bad, None) == ftg.FT_ERR_INVALID
        assert b"share memory" in lib.ft_gemm_last_error()
        kv = sv.FtRows(0x100000, 64, 64, 1)
        a = sv.FtPromptAttentionArgs(fine, kv, kv, bad, None, 0x1000, None, 1, tokens, tokens, 64, 1, 1, 0.0)
        assert lib.ft_prompt_attention_run(a, 0x100000, 1 << 40, 0x1000, None) == ftg.FT_ERR_INVALID
        assert b"share memory" in lib.ft_gemm_last_error()
        cache = _cache(sv, kv_heads=1, token_stride=64)
        t = sv.FtTreeAttentionArgs(fine, bad, None, 0x1000, 0x1000, 0x1000, None, 0, 0, 1, tokens, 4, 4, 0, 0.0)
        assert lib.ft_tree_attention_run(cache, t, 0x100000, 1 << 40, 0x1000, None) == ftg.FT_ERR_INVALID
        assert b"share memory" in lib.ft_gemm_last_error()
    assert refused > 500
    # in place with other strides, and Q and K into one place
    q = sv.FtRows(0x300000, 128, 64, 2)
    assert lib.ft_rotary_run(ctypes.byref(h), q, sv.FtRows(0x300000, 64, 4 * 64, 2), None, None, 0x1000, 4, 1, 0, None) == ftg.FT_ERR_INVALID
    assert lib.ft_rotary_run(ctypes.byref(h), q, sv.FtRows(0x400000, 128, 64, 2), q, sv.FtRows(0x400000, 128, 64, 2), 0x1000, 4, 1, 0, None) == ftg.FT_ERR_INVALID


def test_layers_that_share_memory_are_refused(sv, ftg):
    """Against the definition; pages of one layer between those of another are fine where they do not meet."""
    lib, rng, page, seen = sv._lib(), random.Random(6), 16 * 2 * 64, {True: 0, False: 0}
    cases = [(0, page, 2, 4), (page, page, 2, 4), (3 * page, page, 2, 4), (4 * page, page, 2, 4), (page, 2 * page, 2, 4), (page, 2 * page, 3, 4),
             (page // 2, 2 * page, 2, 1), (0, page, 1, 4), (0, page, 3, 1)]
    for _ in range(2000):
        cases.append((page // 8 * rng.randint(0, 70), page // 8 * rng.randint(8, 70), rng.randint(1, 7), rng.randint(1, 7)))
    for layer_stride, page_stride, layers, pages in cases:
        meet = _share((layer_stride, page_stride), (layers, pages), page)
        cache = _cache(sv, layer_stride=layer_stride, page_stride=page_stride, layers=layers, pages=pages)
        assert (lib.ft_kv_cache_copy_pages(cache, None, None, 0, None) == ftg.FT_ERR_INVALID) == meet, (layer_stride, page_stride, layers, pages)
        seen[meet] += 1
    assert min(seen.values()) > 300


def test_one_slab_as_k_and_v_cannot_be_written(sv, ftg):
    lib, rows, x = sv._lib(), sv.FtRows(0x1000, 128, 64, 2), 0x1000
    both = _cache(sv, v=0x10000)
    assert lib.ft_kv_cache_append(both, 0, rows, rows, x, 1, None, None, None, None, None) == ftg.FT_ERR_INVALID
    assert b"same memory" in lib.ft_gemm_last_error()
    assert lib.ft_kv_cache_accept(both, x, 4, 4, x, x, x, x, 1, x + 64, None) == ftg.FT_ERR_INVALID
    assert b"same memory" in lib.ft_gemm_last_error()
    assert lib.ft_kv_cache_copy_pages(both, None, None, 0, None) == ftg.FT_OK


def test_entry_points_are_seen_only_with_their_types(sv, monkeypatch):
    """While one thread binds, another may call: an entry point without its types would cut addresses to 32 bits."""
    real = sv._lib()

    class Entry:
        def __setattr__(self, name, value):
            assert self not in sv._calls.values(), "published before its types were set"
            object.__setattr__(self, name, value)

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def __getitem__(self, name):
            return Entry()

    library, names = Library(), set(sv._calls)
    monkeypatch.setattr(sv._abi, "load", lambda: library)
    monkeypatch.setattr(sv, "_bound", False)
    monkeypatch.setattr(sv, "_calls", {})
    assert sv._lib() is library
    assert set(sv._calls) == names and all(hasattr(call, "argtypes") for call in sv._calls.values())


def test_threads_that_load_at_once_get_one_library(sv, monkeypatch):
    made = []

    def slow(path):
        time.sleep(0.05)
        made.append(path)
        return unittest.mock.MagicMock()

    monkeypatch.setattr(sv._abi.ctypes, "CDLL", slow)
    monkeypatch.setattr(sv._abi, "_lib", None)
    got = []
    threads = [threading.Thread(target=lambda: got.append(sv._abi.load())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and len(got) == 4 and all(x is got[0] for x in got)


def test_appending_with_closed_rotary_positions_is_refused(sv, ftg):
    """Not K as it is, as if no positions had been given."""
    torch = pytest.importorskip("torch")
    here = types.SimpleNamespace(index=-1)  # where tensors on the host say they are
    cache, rotary = object.__new__(ftg.PagedCache), object.__new__(ftg.Rotary)
    cache.device, cache.dtype, cache.kv_heads, cache.head_dim, cache.address = here, torch.bfloat16, 2, 64, 0
    rotary.device, rotary.head_dim, rotary.handle = here, 64, ctypes.c_void_p()
    k, at = torch.zeros((3, 2, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="closed"):
        cache.append(0, k, k, at, rotary=rotary, positions=at)


def test_numbers_that_leave_their_range_are_refused(sv, ftg):
    """A scale times log2(e), a magnitude in 32 bits, frequencies and a grown base that would be infinite."""
    for bad in (dict(magnitude=1e39), dict(magnitude=-1e39), dict(scaling=1, factor=1e-310), dict(scaling=2, base=1e300, factor=1e300)):
        assert _frequencies(sv, **bad)[0] == ftg.FT_ERR_INVALID, bad
    assert _frequencies(sv, magnitude=3e38)[0] == ftg.FT_OK and _frequencies(sv, scaling=2, base=1e150, factor=1e150)[0] == ftg.FT_OK
    rows = lambda heads: sv.FtRows(0x10000, heads * 128, 128, heads)  # noqa: E731
    for scale, batch, code in ((3e38, 1, ftg.FT_ERR_INVALID), (2.36e38, 1, ftg.FT_ERR_INVALID), (2.3e38, 0, ftg.FT_OK)):
        a = sv.FtPromptAttentionArgs(rows(8), rows(2), rows(2), rows(8), None, 0x1000, None, batch, 16, 16, 128, 1, 1, scale)
        assert sv._lib().ft_prompt_attention_run(a, 0x100000, 1 << 40, 0x1000, None) == code


def test_the_pool_refuses_streams_of_another_device(ftg):
    """Its copies would run on another stream than the caller orders them by; nothing has changed then."""
    torch = pytest.importorskip("torch")
    pool = ftg.PagePool(6, 4)
    free, a = pool.new_sequence(), pool.new_sequence()
    pool.extend([free, a], [3, 6])
    pool.fork(a)
    pool.free(free)  # a hole in front of the used pages, and a last page that two sequences hold
    pool.cache = types.SimpleNamespace(pages=6, page_size=4, device=torch.device("cuda:0"))
    before, other = pool.page_list(a), types.SimpleNamespace(device=torch.device("cuda:1"), cuda_stream=0)
    for call in (lambda: pool.extend([a], [1], stream=other), lambda: pool.compact(stream=other)):
        with pytest.raises(ValueError, match="stream belongs to"):
            call()
        assert pool.page_list(a) == before and pool.length(a) == 6 and pool.free_pages() == 4
