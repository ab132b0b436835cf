"""Threads that share a paged cache, without a GPU: the library's calls are recorded, not made."""
import ctypes
import threading
import time

import pytest
import torch

from syrinx_amd import paged


class _Calls:
    """A library whose attentions take a while, and note whether one came between another's begin and
    end with its workspace."""

    def __init__(self):
        self.busy, self.overlaps, self.made, self.guard = {}, 0, 0, threading.Lock()

    def _attend(self, ws):
        with self.guard:
            self.overlaps += self.busy.get(ws, 0) > 0
            self.busy[ws] = self.busy.get(ws, 0) + 1
            self.made += 1
        time.sleep(0.01)
        with self.guard:
            self.busy[ws] -= 1
        return 0

    def sxq_kv_attention(self, *a):
        return self._attend(a[16])

    def sxq_kv_prefix_attention(self, *a):
        return self._attend(a[17])

    def _need(self, pages, n_q, n_heads, out):
        out._obj.value = paged._COUNTER_BYTES + 64 * n_q
        return 0

    sxq_kv_attention_workspace = sxq_kv_prefix_attention_workspace = _need


def _host_cache():
    """A cache without its constructor, which asks for a GPU: CPU tensors are of device index -1."""
    cache = object.__new__(paged.PagedKvCache)
    vars(cache).update(is8=True, device=torch.device("cpu"), dtype=torch.int8, _index=-1, n_layers=1, n_kv_heads=2, head_dim=64,
                       n_pages=4, page_size=32, max_rows=4, max_len=64, max_blocks=2, _need={}, _ws={}, _lock=threading.Lock(),
                       table=torch.zeros((4, 2), dtype=torch.int32), lens=torch.zeros(4, dtype=torch.int32))
    cache._layer_refs = [ctypes.byref(cache._pages(None, None, None, None))]
    return cache


@pytest.mark.parametrize("prefix", [True, False])
def test_attentions_of_two_threads_do_not_share_a_workspace_at_once(monkeypatch, prefix):
    """An attention of several launches hands over through its workspace: two threads' calls on one
    stream, which both use that stream's, go one after the other (a launch of one between two of the
    other would take its items for its own, whatever their number)."""
    calls = _Calls()
    monkeypatch.setattr(paged, "lib", lambda: calls)
    monkeypatch.setattr(paged, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    cache = _host_cache()
    q = [torch.zeros((n, 4, 64), dtype=torch.bfloat16) for n in (4, 400)]
    rows = [torch.zeros(len(x), dtype=torch.int32) for x in q]

    def work(i):
        for _ in range(5):
            cache.attend(0, q[i], rows=rows[i], pos=rows[i] if prefix else None)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert calls.made == 10 and calls.overlaps == 0
