"""The paged cache without a GPU: every refusal of its C-ABI and of its Python mirror, and the
index arithmetic of its kernels (csrc/sxq_paged.h), enumerated with bad lengths, page ids and
slots: whatever device memory holds, an address stays inside the pool."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from syrinx_amd import SxqError, _lib
from syrinx_amd.paged import KvPages, PagedKvCache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16 = 0, 1, 30


def _pages(dtype=BF16, nkv=2, hd=64, page=16, n_pages=4, k=256, v=256, strides=None):
    ps, hs, os_ = strides or (nkv * page * hd, page * hd, hd)
    return KvPages(dtype, nkv, hd, page, n_pages, k, v, ps, hs, os_)


def _err():
    return _lib.lib().sxq_last_error().decode()


BAD_PAGES = [
    (dict(dtype=8), _lib.ERR_DTYPE, "page dtype"),
    (dict(page=8), _lib.ERR_INVALID, "power of two"),
    (dict(page=48), _lib.ERR_INVALID, "power of two"),
    (dict(page=2048), _lib.ERR_INVALID, "power of two"),
    (dict(n_pages=0), _lib.ERR_INVALID, "n_pages"),
    (dict(n_pages=1 << 27), _lib.ERR_INVALID, "n_pages"),
    (dict(nkv=0), _lib.ERR_INVALID, "n_kv_heads"),
    (dict(hd=60), _lib.ERR_SHAPE, "head_dim"),
    (dict(hd=264), _lib.ERR_SHAPE, "head_dim"),
    (dict(strides=(4096, 1024, 60)), _lib.ERR_SHAPE, "strides"),
    (dict(strides=(4096, 1028, 64)), _lib.ERR_SHAPE, "strides"),
    (dict(strides=(-4096, 1024, 64)), _lib.ERR_SHAPE, "strides"),
    (dict(strides=(0, 1024, 64)), _lib.ERR_SHAPE, "strides"),
    (dict(strides=(1 << 32, 1 << 30, 1 << 25)), _lib.ERR_SHAPE, "pos_stride"),
    (dict(k=None), _lib.ERR_INVALID, "null page pool"),
    (dict(v=264), _lib.ERR_INVALID, "16-byte"),
]


@pytest.mark.parametrize("kw,code,text", BAD_PAGES)
def test_bad_pages_are_refused(kw, code, text):
    L, p = _lib.lib(), _pages(**kw)
    r = ctypes.byref(p)
    assert L.sxq_kv_append(0, r, F32, 256, 1 << 20, 1, 4, None, None, 1e-6, None, None, 0, 0, None, 256, None,
                           None) == code
    assert text in _err() and _err().startswith("kv_append")
    assert L.sxq_kv_attention(0, r, BF16, 256, 256, 1, 4, None, 256, 1, 256, 1, 1, 0.1, 256, 256, 256, 1 << 30,
                              None) == code
    assert text in _err() and _err().startswith("kv_attention")


def _append(pages=None, dtype=F32, qkv=256, stride=512, tokens=1, heads=4, cos=None, sin=None, max_pos=0, pos=256,
            slots=256):
    p = pages or _pages()
    return _lib.lib().sxq_kv_append(0, ctypes.byref(p), dtype, qkv, stride, tokens, heads, None, None, 1e-6, cos, sin,
                                    max_pos, 0, pos, slots, None, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=12), _lib.ERR_DTYPE), (dict(tokens=-1), _lib.ERR_INVALID), (dict(heads=0), _lib.ERR_INVALID),
    (dict(heads=1 << 20), _lib.ERR_INVALID), (dict(stride=511), _lib.ERR_SHAPE), (dict(cos=256), _lib.ERR_INVALID),
    (dict(cos=256, sin=256, max_pos=0), _lib.ERR_INVALID), (dict(qkv=None), _lib.ERR_INVALID),
    (dict(slots=None), _lib.ERR_INVALID), (dict(cos=256, sin=256, max_pos=8, pos=None), _lib.ERR_INVALID)])
def test_append_refusals(kw, code):
    assert _append(**kw) == code and _err().startswith("kv_append")


def test_nothing_to_do_needs_no_gpu():
    assert _append(tokens=0, qkv=None, slots=None, pages=_pages(k=None, v=None)) == _lib.OK
    assert _attend(n_q=0, q=None, pages=_pages(k=None, v=None)) == _lib.OK


def _attend(pages=None, dtype=BF16, q=256, q_stride=256, n_q=1, heads=4, lens=256, n_rows=4, table=256, table_stride=8,
            blocks=8, scale=0.125, out=256, out_stride=256, ws=256, ws_bytes=1 << 40, rows=None):
    p = pages or _pages()
    return _lib.lib().sxq_kv_attention(0, ctypes.byref(p), dtype, q, q_stride, n_q, heads, rows, lens, n_rows, table,
                                       table_stride, blocks, scale, out, out_stride, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=F16), _lib.ERR_DTYPE), (dict(pages=_pages(dtype=F16), dtype=F32), _lib.ERR_DTYPE),
    (dict(pages=_pages(dtype=F32), dtype=BF16), _lib.ERR_DTYPE), (dict(dtype=8), _lib.ERR_DTYPE),
    (dict(heads=3), _lib.ERR_SHAPE), (dict(heads=0), _lib.ERR_SHAPE), (dict(n_q=-1), _lib.ERR_SHAPE),
    (dict(n_q=(1 << 20) + 1), _lib.ERR_SHAPE), (dict(q_stride=248), _lib.ERR_SHAPE),
    (dict(q_stride=260), _lib.ERR_SHAPE), (dict(out_stride=260), _lib.ERR_SHAPE), (dict(n_q=5), _lib.ERR_SHAPE),
    (dict(n_rows=0), _lib.ERR_INVALID), (dict(blocks=0), _lib.ERR_INVALID), (dict(table_stride=7), _lib.ERR_INVALID),
    (dict(blocks=1 << 27, table_stride=1 << 27), _lib.ERR_INVALID),
    (dict(blocks=1 << 26, table_stride=1 << 26, n_q=64, n_rows=64), _lib.ERR_INVALID), (dict(scale=float("inf")), _lib.ERR_INVALID),
    (dict(scale=float("nan")), _lib.ERR_INVALID), (dict(q=None), _lib.ERR_INVALID), (dict(lens=None), _lib.ERR_INVALID),
    (dict(table=None), _lib.ERR_INVALID), (dict(out=None), _lib.ERR_INVALID), (dict(ws=None), _lib.ERR_INVALID),
    (dict(q=264), _lib.ERR_INVALID), (dict(out=8), _lib.ERR_INVALID), (dict(ws=128), _lib.ERR_INVALID),
    (dict(ws_bytes=0), _lib.ERR_INVALID)])
def test_attention_refusals(kw, code):
    assert _attend(**kw) == code and _err().startswith("kv_attention")


def _reserve(page=16, n_pages=4, n_rows=2, blocks=8, stride=8, capacity=4, null=()):
    a = {k: None if k in null else 256 for k in ("add", "lens", "table", "free", "count", "cu", "slots", "pos", "rows",
                                                 "status")}
    return _lib.lib().sxq_kv_reserve(0, page, n_pages, n_rows, blocks, a["add"], a["lens"], a["table"], stride, a["free"],
                                     a["count"], capacity, a["cu"], a["slots"], a["pos"], a["rows"], a["status"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(page=24), _lib.ERR_INVALID), (dict(n_pages=0), _lib.ERR_INVALID), (dict(n_pages=1 << 28), _lib.ERR_INVALID),
    (dict(n_rows=0), _lib.ERR_INVALID), (dict(blocks=0), _lib.ERR_INVALID), (dict(stride=7), _lib.ERR_SHAPE),
    (dict(n_rows=1 << 20, blocks=1 << 12, stride=1 << 12), _lib.ERR_INVALID), (dict(capacity=-1), _lib.ERR_INVALID),
    (dict(capacity=(1 << 30) + 1), _lib.ERR_INVALID),
] + [(dict(null=(k,)), _lib.ERR_INVALID) for k in ("add", "lens", "table", "free", "count", "cu", "slots", "pos", "rows",
                                                     "status")])
def test_reserve_refusals(kw, code):
    assert _reserve(**kw) == code and _err().startswith("kv_reserve")


def test_workspace_refusals():
    L, size = _lib.lib(), ctypes.c_size_t()
    p = _pages(k=None, v=None)  # the size needs no pools
    assert L.sxq_kv_attention_workspace(ctypes.byref(p), 4, 4, None) == _lib.ERR_INVALID
    assert L.sxq_kv_attention_workspace(None, 4, 4, ctypes.byref(size)) == _lib.ERR_INVALID
    assert L.sxq_kv_attention_workspace(ctypes.byref(p), 4, 3, ctypes.byref(size)) == _lib.ERR_SHAPE
    assert L.sxq_kv_attention_workspace(ctypes.byref(p), 4, 4, ctypes.byref(size)) == _lib.OK and size.value > 0
    # a workspace serves any call of no more queries times heads
    last = 0
    for n in (1, 2, 7, 16, 100, 3000, 1 << 20):
        assert L.sxq_kv_attention_workspace(ctypes.byref(p), n, 4, ctypes.byref(size)) == _lib.OK
        assert size.value >= last
        last = size.value


@pytest.mark.parametrize("kw,err", [
    (dict(dtype=torch.int8), ValueError), (dict(max_rows=0), ValueError), (dict(max_len=0), ValueError),
    (dict(device="cpu"), ValueError), (dict(page_size=20), SxqError), (dict(n_pages=0), SxqError)])
def test_python_constructor_refusals(kw, err):
    base = dict(n_pages=4, page_size=16, max_rows=2, max_len=64, device="cpu")
    base.update(kw)
    with pytest.raises(err):
        PagedKvCache(1, 2, 64, **base)


DRIVER = r"""
#include <cstdio>
#include <initializer_list>
#include "sxq_paged.h"
using namespace sxq;
#define EXPECT(c) do { if (!(c)) { std::printf("failed: %s\n", #c); return 1; } } while (0)

int main() {
    const int ints[] = {-2147483647 - 1, -1000, -1, 0, 1, 15, 16, 17, 1023, 1024, 65535, 1 << 24, 2147483646, 2147483647};
    for (int shift = 4; shift <= 10; ++shift)
        for (int blocks : {1, 2, 1000, (int)((1ll << 31) - 1) >> shift}) {
            for (int len : ints) {
                const int c = kv_clamp_len(len, blocks, shift);
                EXPECT(c >= 0 && (int64_t)c <= (int64_t)blocks << shift);
                EXPECT(len < 0 || (int64_t)len > (int64_t)blocks << shift || c == len);
                // every position below the length has a table entry
                EXPECT(kv_blocks(c, shift) <= blocks && (c == 0 || (c - 1) >> shift < kv_blocks(c, shift)));
            }
            const int n_pages = blocks;
            for (int id : ints)
                for (int pos : ints) {
                    const int s = kv_slot(id, pos, shift, n_pages);
                    EXPECT(kv_page_ok(id, n_pages) == (id >= 0 && id < n_pages));
                    EXPECT(s == -1 || (s >= 0 && (int64_t)s < (int64_t)n_pages << shift && s >> shift == id));
                    EXPECT((s == -1) == !kv_page_ok(id, n_pages));
                }
        }
    // the last element of the last slot of a pool whose offsets pass 32 bits
    KvPool p{nullptr, nullptr, 8 * 16 * 128, 16 * 128, 128, 30, 8, 128, 16, 4, 1 << 20};
    EXPECT(kv_slot_base(p, (1 << 24) - 1, 7) + 128 == (int64_t)(1 << 20) * p.page_stride);
    EXPECT(kv_slot_base(p, 0, 0) == 0 && kv_slot_base(p, 17, 3) == p.page_stride + 3 * p.head_stride + 128);
    std::printf("ok\n");
}
"""


def test_index_arithmetic_stays_in_range(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not installed")
    src, exe = tmp_path / "idx.cpp", tmp_path / "idx"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "syrinx_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
