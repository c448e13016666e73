"""GPU tests of ``ChunkedKVCache``: steps with ragged chunks against plain 64-bit attention
over the positions that each head's slots still hold, across evictions and releases."""
import pytest
import torch

from llama3_8b_attention_optimize_b200 import kernels
from llama3_8b_attention_optimize_b200.session import ChunkedKVCache

pytestmark = pytest.mark.gpu
D = 128


def rotate64(x, pos, inv, interleaved):
    """x [n, H, 128] rotated in 64 bits, rounded to bf16 as the cache holds it."""
    y, rot = x.double().clone(), 2 * inv.numel()
    ang = pos.double()[:, None, None] * inv
    c, s = ang.cos(), ang.sin()
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + (1 if interleaved else rot // 2)
    a, b = x[..., ia].double(), x[..., ib].double()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y.to(torch.bfloat16).double()


@pytest.mark.parametrize("interleaved,rot,Hq,Hkv,page,rope", [
    (False, 128, 32, 8, 64, {}),
    (True, 64, 6, 2, 16, dict(scaling="llama3", factor=8.0)),
])
def test_steps_with_eviction(interleaved, rot, Hq, Hkv, page, rope):
    """Tolerance: q and k each rounded to bf16 after a rotation that may differ in its last
    fp32 bit from the 64-bit one, so a score can move by 2 x 2^-8 of sum |q_i k_i| scale on single
    values; over 128 of them that stays below 2^-6 of the scores' spread.  Outputs are held to
    3e-2 absolute, values of unit scale, and to 3e-3 on average."""
    B, G = 3, Hq // Hkv
    cache = ChunkedKVCache(B, num_pages=3 * 700 // page, max_pages_per_seq=640 // page, Hkv=Hkv, Hq=Hq, page_size=page,
                           max_positions=4096, rot_dim=rot, interleaved=interleaved, rope=rope)
    inv = kernels.rope_inv_freq(rot, **rope)[0].cuda()
    gen = torch.Generator("cuda").manual_seed(3)
    total_pages = cache.free_pages
    ks, vs = [[] for _ in range(B)], [[] for _ in range(B)]  # every token's key (rotated) and value, by position
    steps = [[300, 7, 0], [1, 1, 0], [40, 0, 5], "evict", [1, 1, 1], [130, 2, 64], "evict", [1, 0, 1], [33, 3, 1]]
    for new in steps:
        if new == "evict":
            before = [cache.seq_len(b) for b in range(B)]
            cache.evict(128, recent=16, sink=4)
            assert [cache.seq_len(b) for b in range(B)] == [min(n, 128) for n in before]
            assert cache.free_pages == total_pages - sum(-(-cache.seq_len(b) // page) for b in range(B))
            for b in range(B):
                n = cache.seq_len(b)
                for h in range(Hkv):
                    pos = cache.slot_pos[b, h, :n].tolist()
                    assert len(set(pos)) == n
                    if before[b] > 128:  # what is protected stayed
                        last = cache.next_pos(b)
                        assert set(range(4)) | set(range(last - 16, last)) <= set(pos)
            continue
        T = sum(new)
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=gen, device="cuda").to(torch.bfloat16)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        first = [cache.next_pos(b) for b in range(B)]
        out = cache.step(q, k, v, new)
        kernels.device_check()
        t = 0
        for b, n in enumerate(new):
            pos = torch.arange(first[b], first[b] + n, device="cuda")
            assert cache.next_pos(b) == first[b] + n
            if n == 0:
                continue
            ks[b].append(rotate64(k[t:t + n], pos, inv, interleaved))
            vs[b].append(v[t:t + n].double())
            kb, vb = torch.cat(ks[b]), torch.cat(vs[b])
            qb = rotate64(q[t:t + n], pos, inv, interleaved)
            L = cache.seq_len(b)
            for h in range(Hkv):
                held = cache.slot_pos[b, h, :L].long()
                s = torch.einsum("ngd,ld->ngl", qb[:, h * G:(h + 1) * G], kb[held, h]) * D ** -0.5
                s = s.masked_fill((torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None])[:, None],
                                  -torch.inf)
                ref = s.softmax(-1) @ vb[held, h]
                err = (out[t:t + n, h * G:(h + 1) * G].double() - ref).abs()
                assert err.max() <= 3e-2 and err.mean() <= 3e-3, (err.max().item(), err.mean().item())
            t += n
        # the weights handed out in this step, all rows' sum, went to slots that are held
        assert torch.isfinite(cache.acc).all()
    cache.release(0)
    assert cache.seq_len(0) == 0 and cache.next_pos(0) == 0
    out = cache.step(q[:2], k[:2], v[:2], [1, 1, 0])
    want = v[0].repeat_interleave(G, 0)  # a single token attends itself
    assert torch.equal(out[0], want)
    kernels.device_check()


def test_weights_add_up():
    """Every query row hands out weight 1 per head: what the slots received adds up."""
    cache = ChunkedKVCache(2, 64, 16, page_size=64)
    gen = torch.Generator("cuda").manual_seed(1)
    rows = [0, 0]
    for new in ([100, 3], [1, 1], [70, 200]):
        x = torch.randn(sum(new), 48, D, generator=gen, device="cuda").to(torch.bfloat16)
        cache.step(x[:, :32], x[:, 32:40], x[:, 40:], new)
        rows = [r + n for r, n in zip(rows, new)]
    for b in range(2):
        total = cache.acc[b, :, :cache.seq_len(b)].double().sum(-1)
        assert torch.allclose(total, torch.full_like(total, 4.0 * rows[b]), rtol=1e-5)


def test_refusals():
    cache = ChunkedKVCache(2, 4, 4, Hkv=2, Hq=8, page_size=16, max_positions=40)
    x = torch.zeros(60, 12, D, dtype=torch.bfloat16, device="cuda")
    call = lambda new: cache.step(x[:sum(new), :8], x[:sum(new), 8:10], x[:sum(new), 10:], new)  # noqa: E731
    with pytest.raises(ValueError, match="per sequence"):
        call([1])
    with pytest.raises(ValueError, match="rotary table"):
        call([41, 0])
    with pytest.raises(RuntimeError, match="out of pages"):
        call([33, 17])
    assert cache.free_pages == 4  # nothing was taken
    with pytest.raises(ValueError, match="tokens"):
        cache.step(x[:3, :8], x[:2, 8:10], x[:2, 10:], [2, 0])
    call([33, 10])
    with pytest.raises(ValueError):
        cache.evict(0)
    with pytest.raises(ValueError):
        cache.evict(100, recent=80, sink=30)
    cache.evict(20, recent=4)
    assert [cache.seq_len(b) for b in range(2)] == [20, 10] and cache.free_pages == 1
    with pytest.raises(ValueError, match="track_weights"):
        ChunkedKVCache(1, 2, 2, page_size=16, track_weights=False).evict(4)
    with pytest.raises(ValueError):
        ChunkedKVCache(1, 2, 2, page_size=24)
    kernels.device_check()


def test_evictions_keep_the_heaviest():
    """A 64-bit sum of the weight that each position of each head received, kept by position: the
    cache's sums follow it through evictions and reused slots, and what an eviction drops weighs
    no more than any unprotected position that it keeps.

    Tolerance 2^-13 of a sum: a weight's score and lse are each off by 2^-20 sum |q_i k_i| scale,
    below 2^-16 here, the exponential by 2^-18, and up to 1100 fp32 terms enter the sums, 2^-24 each."""
    B, Hq, Hkv, page, budget = 3, 8, 2, 16, 96
    G, M = Hq // Hkv, 1024
    cache = ChunkedKVCache(B, num_pages=90, max_pages_per_seq=30, Hkv=Hkv, Hq=Hq, page_size=page, max_positions=M)
    gen = torch.Generator("cuda").manual_seed(7)
    keys = torch.zeros(B, Hkv, M, D, dtype=torch.float64, device="cuda")
    weight = torch.zeros(B, Hkv, M, dtype=torch.float64, device="cuda")
    dropped = 0
    for new in ([200, 9, 0], [1, 1, 0], "evict", [30, 1, 120], [1, 1, 1], "evict", [1, 0, 1], "evict", [64, 150, 1], "evict", [2, 1, 1]):
        if new == "evict":
            before = [[cache.slot_pos[b, h, :cache.seq_len(b)].tolist() for h in range(Hkv)] for b in range(B)]
            cache.evict(budget, recent=8, sink=2)
            kernels.device_check()
            for b in range(B):
                for h in range(Hkv):
                    kept = set(cache.slot_pos[b, h, :cache.seq_len(b)].tolist())
                    gone = set(before[b][h]) - kept
                    assert kept <= set(before[b][h]) and len(kept) == min(len(before[b][h]), budget)
                    free = [p for p in kept if 2 <= p < cache.next_pos(b) - 8]
                    if gone:
                        w = weight[b, h]
                        assert w[free].min() >= w[sorted(gone)].max() * (1 - 2.0 ** -12)
                    dropped += len(gone)
        else:
            T = sum(new)
            x = torch.randn(T, Hq + 2 * Hkv, D, generator=gen, device="cuda").to(torch.bfloat16)
            pos = torch.cat([torch.arange(cache.next_pos(b), cache.next_pos(b) + n, device="cuda") for b, n in enumerate(new)])
            rot = kernels.rope_positions(x[:, :Hq + Hkv], pos.to(torch.int32), cache.cos, cache.sin).double()
            held = [[cache.slot_pos[b, h, :cache.seq_len(b)].long() for h in range(Hkv)] for b in range(B)]
            cache.step(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], new)
            kernels.device_check()
            t = 0
            for b, n in enumerate(new):
                for h in range(Hkv if n else 0):
                    mine = pos[t:t + n]
                    keys[b, h, mine] = rot[t:t + n, Hq + h]
                    at = torch.cat([held[b][h], mine])
                    s = torch.einsum("ngd,ld->ngl", rot[t:t + n, h * G:(h + 1) * G], keys[b, h, at]) * D ** -0.5
                    L = at.numel()
                    unseen = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
                    weight[b, h, at] += s.masked_fill(unseen[:, None], -torch.inf).softmax(-1).sum((0, 1))
                t += n
        for b in range(B):
            for h in range(Hkv):
                L = cache.seq_len(b)
                want = weight[b, h, cache.slot_pos[b, h, :L].long()]
                assert ((cache.acc[b, h, :L].double() - want).abs() <= 2.0 ** -13 * want).all()
    assert dropped > 300
