"""Host bookkeeping of ``ChunkedKVCache`` without a GPU: the kernels are replaced by stubs
that record what they are given."""
import pytest
import torch

from llama3_8b_attention_optimize_b200 import kernels
from llama3_8b_attention_optimize_b200.session import ChunkedKVCache

D = 128


class Stubs:
    """What reached the kernels; ``fail`` names the one that raises."""

    def __init__(self, monkeypatch):
        self.fail, self.seen = None, {}
        for name in ("kv_extend", "attend_chunk", "attn_weight_sums", "kv_evict"):
            monkeypatch.setattr(kernels, name, getattr(self, name))
        monkeypatch.setattr(kernels, "rope_table", lambda rows, rot, theta, device, **kw: (torch.zeros(rows, rot // 2),) * 2)
        monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)

    def _called(self, name, **what):
        self.seen[name] = {k: v.tolist() for k, v in what.items()}
        if self.fail == name:
            raise torch.OutOfMemoryError(name)

    def kv_extend(self, k, v, kp, vp, table, q_start, lens, positions, cos, sin, *, q, interleaved, slot_pos):
        self._called("kv_extend", table=table, q_start=q_start, lens=lens, positions=positions)
        return q

    def attend_chunk(self, q, kp, vp, table, q_start, lens, *, max_q_len, out, lse):
        self._called("attend_chunk", table=table, q_start=q_start, lens=lens)
        return q

    def attn_weight_sums(self, q, kp, table, q_start, lens, lse, acc, *, max_q_len):
        self._called("attn_weight_sums", table=table, q_start=q_start, lens=lens)

    def kv_evict(self, kp, vp, table, lens, acc, slot_pos, next_pos, budget, *, recent, sink):
        self._called("kv_evict", table=table, lens=lens, next_pos=next_pos)
        lens.clamp_(max=budget)


def step(cache, new):
    x = torch.zeros(sum(new), cache.Hq + 2 * cache.Hkv, D, dtype=torch.bfloat16)
    return cache.step(x[:, :cache.Hq], x[:, cache.Hq:cache.Hq + cache.Hkv], x[:, cache.Hq + cache.Hkv:], new)


@pytest.mark.parametrize("where", ["kv_extend", "attend_chunk", "attn_weight_sums"])
def test_a_step_that_raises_changes_nothing(monkeypatch, where):
    """Lengths, positions and pages stay as they were, on the device too, so that an eviction
    (what a server does when memory runs out) and the next step go by real slots only."""
    stubs = Stubs(monkeypatch)
    cache = ChunkedKVCache(2, num_pages=40, max_pages_per_seq=20, Hkv=1, Hq=4, page_size=16, device="cpu")
    step(cache, [100, 20])
    free, table = cache.free_pages, cache.table.tolist()
    stubs.fail = where
    with pytest.raises(torch.OutOfMemoryError):
        step(cache, [50, 1])
    stubs.fail = None
    assert cache.lens.tolist() == [100, 20] == [cache.seq_len(b) for b in range(2)]
    assert [cache.next_pos(b) for b in range(2)] == [100, 20]
    assert cache.free_pages == free and cache.table.tolist() == table
    cache.evict(64, sink=4)
    assert stubs.seen["kv_evict"]["lens"] == [100, 20] and stubs.seen["kv_evict"]["next_pos"] == [100, 20]
    assert cache.lens.tolist() == [64, 20] == [cache.seq_len(b) for b in range(2)]
    step(cache, [1, 0])
    assert stubs.seen["attend_chunk"]["lens"] == [65, 20] and stubs.seen["kv_extend"]["positions"] == [100]
    assert cache.lens.tolist() == [65, 20]


def test_pages_reserved_ahead_stay_reserved_when_a_step_raises(monkeypatch):
    stubs = Stubs(monkeypatch)
    cache = ChunkedKVCache(2, num_pages=10, max_pages_per_seq=5, Hkv=1, Hq=4, page_size=16, device="cpu")
    cache.reserve([40, 0])
    assert cache.free_pages == 7
    stubs.fail = "attend_chunk"
    with pytest.raises(torch.OutOfMemoryError):
        step(cache, [50, 17])
    assert cache.free_pages == 7
    held = {p for row in cache.table.tolist() for p in row if p >= 0}
    stubs.fail = None
    step(cache, [80, 80])
    pages = [p for row in cache.table.tolist() for p in row]
    assert sorted(pages) == list(range(10)) and held <= set(pages[:5]) and cache.free_pages == 0
