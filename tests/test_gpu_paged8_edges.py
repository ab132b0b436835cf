"""The 8-bit paged cache on the GPU where it can go wrong beside test_gpu_paged8's cases: threads, maps
of more entries than tokens, value scales far from one, pools of other strides under many rows."""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

from syrinx_amd.paged import PagedKvCache, SlotMap
from test_gpu_paged import DT, F64, U32, _close
from test_gpu_paged8 import CT, PREFIX_SPLIT, B, _attend, _cache, _filled, _queries, _reference, cuda  # noqa: F401

pytestmark = pytest.mark.gpu


def _i32(cuda, v):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def test_threads_attend_on_one_stream_at_once(cuda):
    """Two threads, calls of unlike sizes, both on the default stream: each call's outputs are its own."""
    cache, g = _filled(cuda, 2, 64, 16, [5000, 300], "i8", 2)
    calls = []
    for n in (3, 700):
        q = _queries(g, cuda, n, 8, 64, "bf16")
        rows, pos = _i32(cuda, [i % 2 for i in range(n)]), _i32(cuda, [299 - i % 290 for i in range(n)])
        calls.append((q, rows, pos, cache.attend(0, q, rows=rows, pos=pos), cache.attend(0, q, rows=rows)))
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        q, rows, pos = calls[i][:3]
        for _ in range(50):
            got[i].append((cache.attend(0, q, rows=rows, pos=pos), cache.attend(0, q, rows=rows)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 50
        assert all(torch.equal(x, calls[i][3]) and torch.equal(y, calls[i][4]) for x, y in got[i])
