"""The 8-bit paged cache without a GPU: the refusals of its C-ABI (8-bit pages in the calls that
other pages have, the read, the attention over prefixes), and its scales' index arithmetic."""
import ctypes
import os
import shutil
import subprocess

import pytest

from syrinx_amd import _lib
from syrinx_amd.paged import SCALE_BLOCK, KvPages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, I8, BF16, E4M3 = 0, 1, 24, 30, 0x101


def _pages(dtype=I8, nkv=2, hd=64, page=32, n_pages=4, k=256, v=256, strides=None, ks=256, vs=256, scales=None):
    ps, hs, os_ = strides or (nkv * page * hd, page * hd, hd)
    sp, sh = scales or (nkv * page // SCALE_BLOCK, page // SCALE_BLOCK)
    return KvPages(dtype, nkv, hd, page, n_pages, k, v, ps, hs, os_, ks, vs, sp, sh)


def _err():
    return _lib.lib().sxq_last_error().decode()


def _append(pages=None, dtype=F32, qkv=256, stride=1024, tokens=1, heads=4, slots=256):
    p = pages or _pages()
    return _lib.lib().sxq_kv_append(0, ctypes.byref(p), dtype, qkv, stride, tokens, heads, None, None, 1e-6, None, None, 0,
                                    0, None, slots, None, None)


def _attend(pages=None, dtype=BF16, q=256, q_stride=256, n_q=1, heads=4, rows=256, pos=256, lens=256, n_rows=4, table=256,
            table_stride=8, blocks=8, scale=0.125, out=256, out_stride=256, ws=256, ws_bytes=1 << 40, prefix=True):
    p, L = pages or _pages(), _lib.lib()
    if not prefix:
        return L.sxq_kv_attention(0, ctypes.byref(p), dtype, q, q_stride, n_q, heads, rows, lens, n_rows, table, table_stride,
                                  blocks, scale, out, out_stride, ws, ws_bytes, None)
    return L.sxq_kv_prefix_attention(0, ctypes.byref(p), dtype, q, q_stride, n_q, heads, rows, pos, lens, n_rows, table,
                                     table_stride, blocks, scale, out, out_stride, ws, ws_bytes, None)


def _read(pages=None, cu=256, rows=256, start=256, n=2, total=4, lens=256, n_rows=4, table=256, table_stride=8, blocks=8,
          dtype=BF16, k=256, v=256, stride=128):
    p = pages or _pages()
    return _lib.lib().sxq_kv_read(0, ctypes.byref(p), cu, rows, start, n, total, lens, n_rows, table, table_stride, blocks, dtype,
                                  k, v, stride, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=9), _lib.ERR_DTYPE, "page dtype"), (dict(hd=72), _lib.ERR_SHAPE, "multiple of 16"),
    (dict(hd=8), _lib.ERR_SHAPE, "multiple of 16"), (dict(hd=272), _lib.ERR_SHAPE, "head_dim"),
    (dict(strides=(4096, 2048, 72)), _lib.ERR_SHAPE, "strides"), (dict(strides=(4096, 2056, 64)), _lib.ERR_SHAPE, "strides"),
    (dict(scales=(4, 1)), _lib.ERR_SHAPE, "scale strides"), (dict(scales=(1, 2)), _lib.ERR_SHAPE, "scale strides"),
    (dict(scales=(-4, 2)), _lib.ERR_SHAPE, "scale strides"), (dict(scales=(1 << 60, 2)), _lib.ERR_SHAPE, "scale strides"),
    (dict(ks=None), _lib.ERR_INVALID, "null scales"), (dict(vs=None), _lib.ERR_INVALID, "null scales"),
    (dict(ks=258), _lib.ERR_INVALID, "4-byte"), (dict(k=None), _lib.ERR_INVALID, "null page pool"),
    (dict(v=264), _lib.ERR_INVALID, "16-byte"), (dict(page=8), _lib.ERR_INVALID, "power of two")])
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_bad_8_bit_pages_are_refused_everywhere(kw, code, text, dtype):
    p = _pages(**{"dtype": dtype, **kw})
    assert _append(pages=p) == code and text in _err() and _err().startswith("kv_append")
    assert _attend(pages=p, prefix=False) == code and text in _err() and _err().startswith("kv_attention")
    assert _attend(pages=p) == code and text in _err() and _err().startswith("kv_prefix_attention")
    assert _read(pages=p) == code and text in _err() and _err().startswith("kv_read")


def test_other_pages_have_no_scales():
    """16- and 32-bit pages as before: the scales' fields are not looked at."""
    p = _pages(dtype=BF16, ks=None, vs=3, scales=(-1, -1))
    assert _append(pages=p, tokens=0) == _lib.OK
    assert _attend(pages=p, n_q=0, prefix=False) == _lib.OK
    assert _read(pages=p, total=0) == _lib.OK


def test_nothing_to_do_needs_no_gpu():
    p = _pages(k=None, v=None, ks=None, vs=None)
    assert _append(pages=p, tokens=0, qkv=None, slots=None) == _lib.OK
    assert _attend(pages=p, n_q=0, q=None, rows=None, pos=None) == _lib.OK
    assert _attend(pages=p, n_q=0, q=None, prefix=False) == _lib.OK
    assert _read(pages=p, total=0, cu=None, k=None, v=None) == _lib.OK


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=8), _lib.ERR_DTYPE), (dict(dtype=I8), _lib.ERR_DTYPE), (dict(heads=3), _lib.ERR_SHAPE),
    (dict(heads=0), _lib.ERR_SHAPE), (dict(n_q=-1), _lib.ERR_SHAPE), (dict(n_q=(1 << 20) + 1), _lib.ERR_SHAPE),
    (dict(q_stride=248), _lib.ERR_SHAPE), (dict(q_stride=260), _lib.ERR_SHAPE), (dict(out_stride=260), _lib.ERR_SHAPE),
    (dict(n_rows=0), _lib.ERR_INVALID), (dict(blocks=0), _lib.ERR_INVALID), (dict(table_stride=7), _lib.ERR_INVALID),
    (dict(blocks=1 << 26, table_stride=1 << 26), _lib.ERR_INVALID), (dict(scale=float("inf")), _lib.ERR_INVALID),
    (dict(scale=float("nan")), _lib.ERR_INVALID), (dict(q=None), _lib.ERR_INVALID), (dict(lens=None), _lib.ERR_INVALID),
    (dict(table=None), _lib.ERR_INVALID), (dict(out=None), _lib.ERR_INVALID), (dict(ws=None), _lib.ERR_INVALID),
    (dict(q=264), _lib.ERR_INVALID), (dict(out=8), _lib.ERR_INVALID), (dict(ws=128), _lib.ERR_INVALID),
    (dict(ws_bytes=0), _lib.ERR_INVALID)])
@pytest.mark.parametrize("prefix", [True, False])
def test_attention_refusals(kw, code, prefix):
    assert _attend(prefix=prefix, **kw) == code
    assert _err().startswith("kv_prefix_attention" if prefix else "kv_attention")


def test_prefix_attention_takes_8_bit_pages_and_a_map():
    for dtype in (F32, F16, BF16):
        assert _attend(pages=_pages(dtype=dtype), dtype=dtype) == _lib.ERR_DTYPE and "pages of dtype" in _err()
    assert _attend(rows=None) == _lib.ERR_INVALID and _attend(pos=None) == _lib.ERR_INVALID


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=8), _lib.ERR_DTYPE), (dict(dtype=E4M3), _lib.ERR_DTYPE), (dict(n=-1), _lib.ERR_INVALID),
    (dict(total=-1), _lib.ERR_INVALID), (dict(total=(1 << 27) + 1), _lib.ERR_INVALID), (dict(stride=120), _lib.ERR_SHAPE),
    (dict(stride=132), _lib.ERR_SHAPE), (dict(stride=1 << 33), _lib.ERR_SHAPE), (dict(n_rows=0), _lib.ERR_INVALID),
    (dict(blocks=0), _lib.ERR_INVALID), (dict(table_stride=7), _lib.ERR_INVALID), (dict(rows=None, n=5), _lib.ERR_SHAPE),
    (dict(cu=None), _lib.ERR_INVALID), (dict(lens=None), _lib.ERR_INVALID), (dict(table=None), _lib.ERR_INVALID),
    (dict(k=None), _lib.ERR_INVALID), (dict(v=None), _lib.ERR_INVALID), (dict(k=264), _lib.ERR_INVALID)])
@pytest.mark.parametrize("pages", [I8, BF16])
def test_read_refusals(kw, code, pages):
    assert _read(pages=_pages(dtype=pages), **kw) == code and _err().startswith("kv_read")


def test_workspaces():
    L, size = _lib.lib(), ctypes.c_size_t()
    for dtype in (I8, E4M3):
        p = _pages(dtype=dtype, k=None, v=None, ks=None, vs=None)
        for ask in (L.sxq_kv_attention_workspace, L.sxq_kv_prefix_attention_workspace):
            assert ask(ctypes.byref(p), 4, 4, None) == _lib.ERR_INVALID
            assert ask(None, 4, 4, ctypes.byref(size)) == _lib.ERR_INVALID
            assert ask(ctypes.byref(p), 4, 3, ctypes.byref(size)) == _lib.ERR_SHAPE
            last = 0
            for n in (1, 2, 7, 16, 100, 3000, 1 << 20):  # good for any call of no more queries
                assert ask(ctypes.byref(p), n, 4, ctypes.byref(size)) == _lib.OK and size.value >= last
                last = size.value
    p = _pages(dtype=BF16)
    assert L.sxq_kv_prefix_attention_workspace(ctypes.byref(p), 4, 4, ctypes.byref(size)) == _lib.ERR_DTYPE


DRIVER = r"""
#include <cstdio>
#include "sxq_paged.h"
using namespace sxq;
#define EXPECT(c) do { if (!(c)) { std::printf("failed: %s\n", #c); return 1; } } while (0)

int main() {
    // every slot of a pool has one scale of its own block, inside the scales' array
    for (int shift = 4; shift <= 10; ++shift) {
        KvPool p{};
        p.page = 1 << shift;
        p.shift = shift;
        p.nkv = 3;
        p.n_pages = 5;
        p.scale_head_stride = p.page / kScaleBlock;
        p.scale_page_stride = p.nkv * p.scale_head_stride;
        for (int h = 0; h < p.nkv; ++h)
            for (int slot = 0; slot < p.n_pages << shift; ++slot) {
                const int64_t at = kv_scale_at(p, slot, h);
                EXPECT(at >= 0 && at < p.n_pages * p.scale_page_stride);
                EXPECT(at == (slot >> shift) * p.scale_page_stride + h * p.scale_head_stride + (slot % p.page) / 16);
            }
    }
    // the last slot there can be, strides that pass 32 bits
    KvPool p{};
    p.page = 16;
    p.shift = 4;
    p.scale_page_stride = (int64_t)1 << 33;
    p.scale_head_stride = 1;
    EXPECT(kv_scale_at(p, 0x7FFFFFEF, 7) == (((int64_t)0x7FFFFFEF >> 4) << 33) + 7);
    std::printf("ok\n");
}
"""


def test_scale_indexes(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not installed")
    src, exe = tmp_path / "idx.cpp", tmp_path / "idx"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "syrinx_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
