"""GPU tests of the operators that serve a paged cache chunk by chunk: rotary positions,
ragged append, chunk attention, accumulated weights and eviction, against plain 64-bit
forms.  Unwritten cache rows hold NaN, block tables name no page past each sequence's length.

Tolerances (u = 2^-8 is a bf16 rounding's relative error, f = 2^-24 an fp32 one's):
  rotation    2^-22 (|a| + |b|) for the table's rounding, two products and a sum; then u |y| in bf16
  score       ds = 2^-20 scale sum |q_i k_i|: 128 fp32 products and sums
  weight      exp of a score off by ds, evaluated to 2^-13 where the weight is rounded to bf16
              anyway, to 2^-20 where it is summed in fp32
  attention   weights rounded to bf16 in numerator and sum: (2 u + 2 ds + 2^-12) sum w |v| + u |o|
  lse         ds + 2^-18 + f (terms) + 2^-22 |lse|
  sums        (ds + 2^-20 + 2^-22 (|s| + |lse|) + f (terms)) sum p + 2^-22 of the total
"""
import math

import numpy as np
import pytest
import torch

from llama3_8b_attention_optimize_b200 import _lib, kernels
from llama3_8b_attention_optimize_b200.kernels import GqaError

pytestmark = pytest.mark.gpu
D = 128
U, F = 2.0 ** -8, 2.0 ** -24


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(*shape, seed, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Batch:
    """A ragged batch over shuffled pages: new[b] tokens of sequence b, lens[b] slots."""

    def __init__(self, new, lens, Hq, Hkv, page, seed=1, scale_q=1.0, spare_pages=0, pad_tokens=0, extra_table=1,
                 pool_pages=None):
        self.new, self.len_list, self.Hq, self.Hkv, self.page = new, lens, Hq, Hkv, page
        self.B, self.T = len(new), sum(new) + pad_tokens
        need = [-(-max(n, 0) // page) for n in lens]
        self.max_pages = max(need + [1]) + extra_table
        self.cap = self.max_pages * page
        pool = (sum(need) + 1 + spare_pages) if pool_pages is None else pool_pages
        order = np.random.default_rng(seed).permutation(pool)
        table = np.full((self.B, self.max_pages), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table_list = table
        self.table = torch.from_numpy(table).cuda()
        self.q_start = i32([sum(new[:b]) for b in range(self.B + 1)])
        self.lens = i32(lens)
        nan = float("nan")
        self.kp = torch.full((pool, Hkv, page, D), nan, dtype=torch.bfloat16, device="cuda")
        self.vp = torch.full_like(self.kp, nan)
        for b, n in enumerate(lens):
            for h in range(Hkv) if n > 0 else ():
                slot = torch.arange(n, device="cuda")
                pages = self.table[b].long()[slot // page]
                self.kp[pages, h, slot % page] = randn(n, D, seed=seed * 7919 + b * 64 + h)
                self.vp[pages, h, slot % page] = randn(n, D, seed=seed * 104729 + b * 64 + h + 1)
        self.q = randn(self.T, Hq, D, seed=seed + 5, scale=scale_q)

    def kv(self, pool, b, h):
        n = self.len_list[b]
        slot = torch.arange(n, device="cuda")
        return pool[self.table[b].long()[slot // self.page], h, slot % self.page].double()

    def scores(self, b, h, causal, scale):
        """q [n, G, D] against the slots of (b, kv head h): scores [n, G, len] (-inf unseen), ds [n, G]."""
        n, L, G = self.new[b], self.len_list[b], self.Hq // self.Hkv
        t0 = sum(self.new[:b])
        q = self.q[t0:t0 + n, h * G:(h + 1) * G].double()
        k = self.kv(self.kp, b, h)
        s = torch.einsum("ngd,ld->ngl", q, k) * scale
        ds = torch.einsum("ngd,ld->ngl", q.abs(), k.abs()).amax(-1) * scale * 2.0 ** -20 if L else torch.zeros(n, G).cuda()
        last = torch.arange(L - n, L, device="cuda") if causal else torch.full((n,), L - 1, device="cuda")
        seen = torch.arange(L, device="cuda")[None] <= last[:, None]
        return s.masked_fill(~seen[:, None], -math.inf), ds

    def check_attend(self, out, lse, causal=True, scale=None):
        scale = D ** -0.5 if scale is None else scale
        G = self.Hq // self.Hkv
        for b in range(self.B):
            n, t0 = self.new[b], sum(self.new[:b])
            if n == 0:
                continue
            for h in range(self.Hkv):
                s, ds = self.scores(b, h, causal, scale)
                norm = s.logsumexp(-1) if self.len_list[b] else torch.full((n, G), -math.inf, dtype=torch.float64).cuda()
                w = torch.where(norm[..., None] == -math.inf, 0.0, (s - norm[..., None]).exp())
                v = self.kv(self.vp, b, h)
                ref, a = w @ v, w @ v.abs()
                got = out[t0:t0 + n, h * G:(h + 1) * G].double()
                bound = (2 * U + 2 * ds[..., None] + 2.0 ** -12) * a + U * ref.abs()
                assert torch.isfinite(got).all()
                worst = ((got - ref).abs() - bound).max().item()
                assert worst <= 0, (b, h, worst)
                if lse is not None:
                    g = lse[t0:t0 + n, h * G:(h + 1) * G].double()
                    empty = norm == -math.inf
                    assert torch.equal(g == -math.inf, empty)
                    tol = ds + 2.0 ** -18 + F * self.len_list[b] + 2.0 ** -22 * norm.abs()
                    assert ((g - norm).abs() <= tol)[~empty].all(), ((g - norm).abs() - tol)[~empty].max()

    def attend(self, **kw):
        return kernels.attend_chunk(self.q, self.kp, self.vp, self.table, self.q_start, self.lens, **kw)


# ------------------------------------------------------------------ rotary positions
def rope_ref(x, positions, inv, mscale, interleaved, inverse):
    """64-bit rotation and, per value, |a| + |b| of its pair."""
    y, mag = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    rot = 2 * inv.numel()
    ang = positions.double()[:, None, None] * inv.cuda()
    c, s = ang.cos() * mscale, ang.sin() * (-mscale if inverse else mscale)
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + (1 if interleaved else rot // 2)
    a, b = x[..., ia].double(), x[..., ib].double()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * mscale
    return y, mag


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,d,rot,scaling", [
    (1, 1, 128, 128, {}),
    (7, 3, 80, 20, dict(scaling="linear", factor=4.0)),        # half a rotation chunk: one value at a time
    (33, 32, 128, 64, dict(scaling="llama3", factor=8.0)),
    (130, 5, 256, 256, dict(scaling="yarn", factor=16.0, original_len=4096)),
    (3, 40, 2, 2, {}),
    (5, 2, 97, 96, {}),
])
def test_rope_positions(dtype, interleaved, T, H, d, rot, scaling):
    rows = 131072
    x = randn(T, H, d, seed=3, dtype=dtype)
    pos = torch.randint(0, rows, (T,), generator=gen(4), device="cuda", dtype=torch.int32)
    pos[0] = rows - 1
    cos, sin = kernels.rope_table(rows, rot, **scaling)
    inv, m = kernels.rope_inv_freq(rot, **scaling)
    for inverse in (False, True):
        y = kernels.rope_positions(x, pos, cos, sin, interleaved=interleaved, inverse=inverse)
        ref, mag = rope_ref(x, pos, inv, m, interleaved, inverse)
        d_fp = 2.0 ** -22 * mag
        bound = d_fp if dtype == torch.float32 else U * (ref.abs() + d_fp) + d_fp
        assert ((y.double() - ref).abs() <= bound).all()
        assert torch.equal(y[..., rot:], x[..., rot:])
    kernels.device_check()


def test_rope_positions_strides_alignment_and_in_place():
    T, H, rows = 19, 6, 64
    cos, sin = kernels.rope_table(rows, 64)
    pos = torch.randint(0, rows, (T,), generator=gen(1), device="cuda", dtype=torch.int32)
    base = randn(T, H + 3, 130, seed=2)
    views = [base[:, 1:1 + H, :128], base[:, 1:1 + H, 1:129],                       # aligned, one value off
             randn(H, T, 128, seed=3).transpose(0, 1),                              # head-major
             randn(T, 1, 128, seed=4).expand(T, H, 128)]                            # one head broadcast
    for x in views:
        want = kernels.rope_positions(x.contiguous(), pos, cos, sin)
        assert torch.equal(kernels.rope_positions(x, pos, cos, sin), want)
        out = torch.full((H, T, 140), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)[..., :128]
        assert torch.equal(kernels.rope_positions(x, pos, cos, sin, out=out), want)
        if x.stride(1):
            assert kernels.rope_positions(x, pos, cos, sin, out=x) is x
            assert torch.equal(x, want)
    kernels.device_check()


def test_rope_gradient_is_the_inverse_rotation():
    """<w, R(x + e d) - R(x - e d)> / 2e = <R^T w, d>, R^T from the kernel's inverse; with yarn's scale too."""
    T, H, d, rot = 40, 4, 96, 48
    cos, sin = kernels.rope_table(5000, rot, scaling="yarn", factor=4.0, original_len=1024)
    pos = torch.randint(0, 5000, (T,), generator=gen(1), device="cuda", dtype=torch.int32)
    for il in (False, True):
        x, w, e = (randn(T, H, d, seed=s, dtype=torch.float32) for s in (5, 6, 7))
        r = lambda z: kernels.rope_positions(z, pos, cos, sin, interleaved=il).double()  # noqa: E731
        lhs = ((w.double() * (r(x + 0.5 * e) - r(x - 0.5 * e))).sum()).item()
        g = kernels.rope_positions(w, pos, cos, sin, interleaved=il, inverse=True).double()
        rhs = (g * e.double()).sum().item()
        mag = (w.double().abs() * (x.double().abs() + e.double().abs())).sum().item()
        assert abs(lhs - rhs) <= 2.0 ** -20 * mag


def test_rope_position_outside_the_table_skips_its_token():
    cos, sin = kernels.rope_table(10, 128)
    x = randn(3, 2, 128, seed=1)
    out = torch.full_like(x, 5.0)
    kernels.rope_positions(x, i32([3, 10, -1]), cos, sin, out=out)
    with pytest.raises(GqaError) as e:
        kernels.device_check()
    assert e.value.code == _lib.GQA_ERR_DEVICE_INPUT
    assert (out[1:] == 5.0).all() and not (out[0] == 5.0).all()
    kernels.device_check()


def test_rope_offsets_past_32_bits():
    T, H = 9, 2
    big = torch.empty(T, 270_000_000, dtype=torch.bfloat16, device="cuda")  # 2.4e9 values
    x = big[:, -H * 128:].unflatten(1, (H, 128))
    x.copy_(randn(T, H, 128, seed=3))
    cos, sin = kernels.rope_table(100, 128)
    pos = i32(list(range(50, 50 + T)))
    want = kernels.rope_positions(x.contiguous(), pos, cos, sin)
    assert torch.equal(kernels.rope_positions(x, pos, cos, sin, out=x), want)


# ------------------------------------------------------------------ ragged append
@pytest.mark.parametrize("page", [1, 16, 48, 128])
@pytest.mark.parametrize("rot,interleaved", [(128, False), (64, True), (20, False), (6, True), (0, False)])
def test_extend(page, rot, interleaved):
    new, lens = [5, 0, 1, 33], [5, 4, 71, 130]
    bt = Batch(new, lens, 8, 2, page, pad_tokens=3)
    T = bt.T
    qkv = randn(T, 12, D, seed=9)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    pos = torch.randint(0, 500, (T,), generator=gen(2), device="cuda", dtype=torch.int32)
    cos, sin = kernels.rope_table(500, rot) if rot else (None, None)
    inv = kernels.rope_inv_freq(rot)[0] if rot else torch.zeros(0, dtype=torch.float64)
    kp0, vp0 = bt.kp.clone(), bt.vp.clone()
    slot_pos = torch.full((4, 2, bt.cap), -7, dtype=torch.int32, device="cuda")
    q_out = torch.full((T, 8, D), 3.0, dtype=torch.bfloat16, device="cuda")
    kernels.kv_extend(k, v, bt.kp, bt.vp, bt.table, bt.q_start, bt.lens, pos, cos, sin, q=q, q_out=q_out,
                      interleaved=interleaved, slot_pos=slot_pos)
    kernels.device_check()

    def near(y, x, p):
        ref, mag = rope_ref(x, p, inv, 1.0, interleaved, False)
        return ((y.double() - ref).abs() <= U * (ref.abs() + 2.0 ** -22 * mag) + 2.0 ** -22 * mag).all()

    n = sum(new)
    assert near(q_out[:n], q[:n], pos[:n]) and (q_out[n:] == 3.0).all()
    touched = torch.zeros(kp0.shape[:3], dtype=torch.bool, device="cuda")
    want_pos = torch.full_like(slot_pos, -7)
    t = 0
    for b in range(4):
        for i in range(new[b]):
            slot = lens[b] - new[b] + i
            page_no, row = int(bt.table_list[b, slot // page]), slot % page
            touched[page_no, :, row] = True
            want_pos[b, :, slot] = pos[t]
            assert near(bt.kp[page_no, :, row][None], k[t][None], pos[t:t + 1])
            assert torch.equal(bt.vp[page_no, :, row], v[t])
            t += 1
    for a, b0 in ((bt.kp, kp0), (bt.vp, vp0)):
        assert torch.equal(a.view(torch.int16)[~touched], b0.view(torch.int16)[~touched])
    assert torch.equal(slot_pos, want_pos)
    # positions default to the slots
    if rot:
        again = torch.empty_like(q_out)
        slots = torch.cat([torch.arange(L - c, L, device="cuda", dtype=torch.int32) for L, c in zip(lens, new)])
        kernels.kv_extend(k, v, bt.kp, bt.vp, bt.table, bt.q_start, bt.lens, None, cos, sin, q=q, q_out=again,
                          interleaved=interleaved)
        assert near(again[:n], q[:n], slots)
    kernels.device_check()


def test_extend_many_tokens_matches_one_sequence_at_a_time():
    new, lens = [1500, 0, 3100, 777], [1500, 10, 4000, 800]  # several tokens a block
    bt = Batch(new, lens, 4, 1, 16, seed=3)
    k, v = randn(bt.T, 1, D, seed=1), randn(bt.T, 1, D, seed=2)
    cos, sin = kernels.rope_table(4096)
    q_out = kernels.kv_extend(k, v, bt.kp, bt.vp, bt.table, bt.q_start, bt.lens, None, cos, sin, q=bt.q)
    for b in range(4):
        if new[b] == 0:
            continue
        sl = slice(sum(new[:b]), sum(new[:b + 1]))
        kp, vp = torch.zeros_like(bt.kp), torch.zeros_like(bt.vp)
        for c in range(0, new[b], 500):  # short calls take one token a block
            sub = slice(sl.start + c, min(sl.stop, sl.start + c + 500))
            one = kernels.kv_extend(k[sub], v[sub], kp, vp, bt.table[b:b + 1], i32([0, sub.stop - sub.start]),
                                    i32([lens[b] - new[b] + c + sub.stop - sub.start]), None, cos, sin, q=bt.q[sub])
            assert torch.equal(one, q_out[sub])
        slot = torch.arange(lens[b] - new[b], lens[b], device="cuda")
        pg = bt.table[b].long()[slot // 16]
        assert torch.equal(kp[pg, :, slot % 16], bt.kp[pg, :, slot % 16])
        assert torch.equal(vp[pg, :, slot % 16], bt.vp[pg, :, slot % 16])
    kernels.device_check()


def test_extend_reports_bad_device_input_and_writes_nothing():
    bt = Batch([2, 2], [4, 4], 4, 1, 16)
    cos, sin = kernels.rope_table(8)
    k = randn(4, 1, D, seed=1)

    def bad(table=bt.table, q_start=bt.q_start, lens=bt.lens, pos=None, skipped=1):
        kp, vp = torch.zeros_like(bt.kp), torch.zeros_like(bt.vp)
        kernels.kv_extend(k, k, kp, vp, table, q_start, lens, pos, cos, sin)
        with pytest.raises(GqaError) as e:
            kernels.device_check()
        assert e.value.code == _lib.GQA_ERR_DEVICE_INPUT
        rows = int((vp != 0).any(-1).sum())
        assert rows == 4 - skipped, rows

    bad(pos=i32([0, 8, 1, 2]))
    bad(pos=i32([0, -1, 1, 2]))
    broken = bt.table.clone()
    broken[1, 0] = bt.kp.shape[0]
    bad(table=broken, skipped=2)
    bad(lens=i32([1, 4]))                     # its first token would lie in slot -1
    bad(lens=i32([4, bt.cap + 1]), pos=i32([0, 1, 2, 3]), skipped=2 if bt.table_list[1, -1] < 0 else 1)
    bad(q_start=i32([1, 2, 4]))


# ------------------------------------------------------------------ chunk attention
SHAPES = [
    # new, lens, Hq, Hkv, page
    ([1], [1], 4, 1, 16),
    ([1, 1, 1], [1, 200, 129], 32, 8, 128),
    ([1, 0, 3, 0], [17, 5, 3, 0], 8, 2, 16),                 # sequences without new tokens, an empty one
    ([7, 130, 1, 64], [7, 430, 1000, 64], 8, 2, 48),         # pages that end inside a tile
    ([257], [257], 8, 8, 64),                                # one query head a kv head
    ([100, 29], [612, 500], 24, 8, 256),                     # three
    ([33], [700], 16, 1, 112),                               # sixteen
    ([65, 2], [1025, 999], 20, 4, 16),                       # five
    ([1] * 40, [1 + 37 * i for i in range(40)], 8, 2, 32),
    ([300, 1, 1], [2300, 1900, 2047], 32, 8, 64),
    ([5], [40], 33, 1, 16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lens,Hq,Hkv,page", SHAPES)
def test_attend(new, lens, Hq, Hkv, page, causal):
    bt = Batch(new, lens, Hq, Hkv, page, pad_tokens=2)
    lse = torch.full((bt.T, Hq), 9.0, device="cuda")
    out = torch.full((bt.T, Hq, D), 9.0, dtype=torch.bfloat16, device="cuda")
    for hint in (0, max(new)):
        bt.attend(causal=causal, max_q_len=hint, out=out, lse=lse)
        kernels.device_check()
        bt.check_attend(out, lse, causal)
        n = sum(new)
        assert (out[n:] == 9.0).all() and (lse[n:] == 9.0).all()  # padding tokens are not written
        assert torch.equal(bt.attend(causal=causal, max_q_len=hint, lse=lse)[:n], out[:n])  # repeats bit for bit
        bt.check_attend(bt.attend(causal=causal, max_q_len=hint), None, causal)


@pytest.mark.parametrize("scale_q", [0.0, 8.0, 40.0])
def test_attend_flat_and_peaked_scores(scale_q):
    bt = Batch([50, 1], [800, 1500], 8, 2, 32, scale_q=scale_q, seed=11)
    lse = torch.empty(bt.T, 8, device="cuda")
    bt.check_attend(bt.attend(lse=lse), lse)
    bt.check_attend(bt.attend(lse=lse, scale=0.01), lse, scale=0.01)


@pytest.mark.parametrize("hint", [0, 1, 1000])
def test_attend_rows_that_see_nothing(hint):
    """More new tokens than slots: the first ones see none (as when a cache was cut below them)."""
    bt = Batch([6, 200, 1, 3], [2, 70, 0, 0], 8, 2, 16)
    lse = torch.empty(bt.T, 8, device="cuda")
    out = bt.attend(lse=lse, max_q_len=hint)
    kernels.device_check()
    bt.check_attend(out, lse)
    assert (out[:4] == 0).all() and (lse[:4] == -math.inf).all() and torch.isfinite(lse[4:6]).all()
    assert (out[6 + 200:] == 0).all()


def test_attend_strides():
    new, lens = [20, 3], [150, 40]
    bt = Batch(new, lens, 8, 2, 16)
    want = bt.attend()
    T = bt.T
    fused = torch.zeros(T, 12, D, dtype=torch.bfloat16, device="cuda")
    fused[:, 2:10] = bt.q
    heads = torch.zeros(8, T + 5, D, dtype=torch.bfloat16, device="cuda")
    heads[:, :T] = bt.q.transpose(0, 1)
    for q in (fused[:, 2:10], heads[:, :T].transpose(0, 1)):
        out = torch.full((8, T, D + 8), 4.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)[..., :D]
        got = kernels.attend_chunk(q, bt.kp, bt.vp, bt.table, bt.q_start, bt.lens, out=out)
        assert torch.equal(got, want)
    same = bt.q[:, :1].expand(T, 8, D)  # one query head broadcast
    ref = kernels.attend_chunk(same.contiguous(), bt.kp, bt.vp, bt.table, bt.q_start, bt.lens)
    assert torch.equal(kernels.attend_chunk(same, bt.kp, bt.vp, bt.table, bt.q_start, bt.lens), ref)
    kernels.device_check()


def test_attend_other_stream_and_repeat():
    bt = Batch([90, 1, 700], [990, 1300, 2000], 32, 8, 128, seed=21)
    want = bt.attend()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bt.attend()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros_like(want)
    ws = torch.empty(max(16, kernels.attend_chunk_workspace_bytes(bt.T, 32, 8)), dtype=torch.uint8, device="cuda")
    with torch.cuda.graph(graph):
        bt.attend(out=out, workspace=ws)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    # a replay follows the lengths on the device
    bt.lens.copy_(i32([500, 40, 700]))
    bt.len_list = [500, 40, 700]
    graph.replay()
    torch.cuda.synchronize()
    bt.check_attend(out, None)


def test_attend_large_pool_offsets():
    """Pages at the far end of a pool of more than 2^31 values, everything else uninitialised."""
    pages = 2200
    bt = Batch([3, 1], [1500, 2000], 32, 8, 1024, pool_pages=5, extra_table=2)
    kp = torch.empty(pages, 8, 1024, D, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    kp[-4:] = randn(4, 8, 1024, D, seed=1)
    vp[-4:] = randn(4, 8, 1024, D, seed=2)
    bt.kp, bt.vp = kp, vp
    bt.table_list = np.array([[pages - 1, pages - 3, -1, -1], [pages - 4, pages - 2, -1, -1]], np.int32)
    bt.table = torch.from_numpy(bt.table_list).cuda()
    lse = torch.empty(bt.T, 32, device="cuda")
    out = bt.attend(lse=lse)
    kernels.device_check()
    bt.check_attend(out, lse)
    acc = torch.zeros(2, 8, bt.cap, device="cuda")
    check_weights(bt, lse, acc, kernels.attn_weight_sums(bt.q, kp, bt.table, bt.q_start, bt.lens, lse, acc.clone()))


def test_attend_matches_the_prefill_and_the_paged_decode():
    """The framework's own kernels on the same problem, each within its own rounding."""
    S = 300
    q, k, v = randn(32, S, D, seed=1), randn(8, S, D, seed=2), randn(8, S, D, seed=3)
    bt = Batch([S], [S], 32, 8, 128)
    bt.q = q.transpose(0, 1)
    kernels.kv_extend(k.transpose(0, 1), v.transpose(0, 1), bt.kp, bt.vp, bt.table, bt.q_start, bt.lens)
    got = bt.attend().transpose(0, 1)
    want = kernels.prefill(q, k, v)
    assert (got.float() - want.float()).abs().max() <= 2e-2
    one = kernels.attend_chunk(q[:, -1][None], bt.kp, bt.vp, bt.table, i32([0, 1]), bt.lens)
    dec = kernels.decode_paged(q[:, -1][None].contiguous(), bt.kp, bt.vp, bt.table, bt.lens)
    assert (one.float() - dec.float()).abs().max() <= 2e-2
    kernels.device_check()


@pytest.mark.parametrize("what", ["page", "length", "q_start", "q_start_end"])
def test_attend_reports_bad_device_input(what):
    bt = Batch([3, 2], [60, 40], 8, 2, 16)
    table, lens, q_start = bt.table.clone(), bt.lens.clone(), bt.q_start.clone()
    if what == "page":
        table[0, 1] = bt.kp.shape[0] + 5
    elif what == "length":
        lens[1] = bt.cap + 1
        table[1] = table[0, 0]
    elif what == "q_start":
        q_start[1] = -2
    else:
        q_start[2] = bt.T + 9
    kernels.attend_chunk(bt.q, bt.kp, bt.vp, table, q_start, lens)
    with pytest.raises(GqaError) as e:
        kernels.device_check()
    assert e.value.code == _lib.GQA_ERR_DEVICE_INPUT
    kernels.device_check()
    bt.check_attend(bt.attend(), None)  # the next call is sound again


@pytest.mark.parametrize("starts", [[0, 5, 0, 5], [0, 3, 9, 5], [-1, 3, 4, 5]])
def test_q_start_out_of_order_computes_nothing(starts):
    """Such sequences could share tokens and have more steps than the host has counted."""
    bt = Batch([3, 1, 1], [60, 40, 300], 8, 2, 16)
    lse = torch.zeros(bt.T, 8, device="cuda")
    out = torch.full_like(bt.q, 7.0).contiguous()
    acc = torch.full((3, 2, bt.cap), 3.0, device="cuda")
    acc_out = torch.full_like(acc, 5.0)
    q_start = i32(starts)
    kernels.attend_chunk(bt.q, bt.kp, bt.vp, bt.table, q_start, bt.lens, out=out)
    with pytest.raises(GqaError) as e:
        kernels.device_check()
    assert e.value.code == _lib.GQA_ERR_DEVICE_INPUT
    kernels.attn_weight_sums(bt.q, bt.kp, bt.table, q_start, bt.lens, lse, acc, acc_out=acc_out)
    with pytest.raises(GqaError) as e:
        kernels.device_check()
    assert e.value.code == _lib.GQA_ERR_DEVICE_INPUT
    assert (out == 7.0).all() and (acc_out == 5.0).all()
    kernels.device_check()


# ------------------------------------------------------------------ accumulated weights
def check_weights(bt, lse, acc, got, causal=True, scale=None):
    scale = D ** -0.5 if scale is None else scale
    G = bt.Hq // bt.Hkv
    for b in range(bt.B):
        n, L, t0 = bt.new[b], bt.len_list[b], sum(bt.new[:b])
        assert torch.equal(got[b, :, L:], acc[b, :, L:])
        for h in range(bt.Hkv) if L else ():
            base = acc[b, h, :L].double().clone()
            base[max(L - n, 0):] = 0.0
            p, err = torch.zeros(L, dtype=torch.float64, device="cuda"), 0.0
            if n:
                s, ds = bt.scores(b, h, causal, scale)
                ln = lse[t0:t0 + n, h * G:(h + 1) * G].double()
                ok = ln != -math.inf
                p = torch.where(ok[..., None], (s - ln[..., None]).exp(), 0.0).sum((0, 1))
                mag = s.masked_fill(s == -math.inf, 0.0).abs().max().item() + ln[ok].abs().max().item() if ok.any() else 0.0
                err = ds.max().item() + 2.0 ** -20 + 2.0 ** -22 * mag + F * n * G
            total = base + p
            assert ((got[b, h, :L].double() - total).abs() <= err * p + 2.0 ** -22 * total.abs()).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lens,Hq,Hkv,page", SHAPES)
def test_weight_sums(new, lens, Hq, Hkv, page, causal):
    bt = Batch(new, lens, Hq, Hkv, page, pad_tokens=1)
    lse = torch.empty(bt.T, Hq, device="cuda")
    bt.attend(causal=causal, lse=lse)
    acc = torch.rand(bt.B, Hkv, bt.cap, generator=gen(8), device="cuda")
    for hint in (0, max(new)):
        out = acc.clone()
        got = kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc, causal=causal, max_q_len=hint,
                                       acc_out=out)
        assert got is out
        kernels.device_check()
        check_weights(bt, lse, acc, got, causal)
        inplace = acc.clone()
        kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, inplace, causal=causal, max_q_len=hint)
        assert torch.equal(inplace, got)


def test_weight_sums_rows_that_see_nothing_and_total():
    bt = Batch([6, 40, 1], [2, 300, 77], 8, 2, 16, seed=31)
    lse = torch.empty(bt.T, 8, device="cuda")
    bt.attend(lse=lse)
    acc = torch.zeros(3, 2, bt.cap, device="cuda")
    got = kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc.clone())
    check_weights(bt, lse, acc, got)
    # every row that sees a slot hands out weight 1
    assert torch.allclose(got[1].sum(-1), torch.full((2,), 160.0, device="cuda"), rtol=1e-5)
    assert torch.allclose(got[2].sum(-1), torch.full((2,), 4.0, device="cuda"), rtol=1e-5)


def test_weight_sums_strided_queries_and_streams():
    bt = Batch([20, 3, 1], [150, 40, 600], 8, 2, 16, scale_q=4.0)
    lse = torch.empty(bt.T, 8, device="cuda")
    bt.attend(lse=lse)
    acc = torch.zeros(3, 2, bt.cap, device="cuda")
    want = kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc.clone())
    check_weights(bt, lse, acc, want)
    heads = bt.q.transpose(0, 1).contiguous().transpose(0, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.attn_weight_sums(heads, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc, acc_out=acc.clone())
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("new,ctx,causal", [(1, 8191, True), (1, 1500, True), (24, 4000, True), (300, 3000, True),
                                            (3, 5000, False)])
def test_busy_memory_changes_no_result(new, ctx, causal):
    """Loads land late and out of order while DRAM is busy: every call gives the quiet call's bits."""
    rng = np.random.default_rng(new + ctx)
    B = 48 if new < 16 else 6
    lens = [int(rng.integers(max(new, ctx // 32), ctx + 1)) for _ in range(B)]
    bt = Batch([new] * B, lens, 32, 8, 128, seed=3)
    lse = torch.empty(bt.T, 32, device="cuda")
    acc = torch.rand(B, 8, bt.cap, generator=gen(4), device="cuda")
    traffic = torch.empty(1 << 26, device="cuda")
    out = bt.attend(causal=causal, lse=lse).clone()
    sums = kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc, causal=causal, acc_out=acc.clone())
    torch.cuda.synchronize()
    lse_out = torch.empty_like(lse)
    for i in range(60):
        traffic.fill_(i)  # its writes go on in DRAM while the next kernel starts
        got = bt.attend(causal=causal, lse=lse_out)
        assert torch.equal(got, out) and torch.equal(lse_out, lse)
        traffic.fill_(-i)
        got = kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc, causal=causal,
                                       acc_out=acc.clone())
        assert torch.equal(got, sums)
    kernels.device_check()


# ------------------------------------------------------------------ eviction
def evict_ref(bt, acc, slot_pos, next_pos, budget, recent, sink):
    """Plain form on the host: (kp, vp, acc, slot_pos, lens) after the cut."""
    kp, vp = bt.kp.view(torch.int16).cpu().numpy().copy(), bt.vp.view(torch.int16).cpu().numpy().copy()
    a, s = acc.cpu().numpy().copy(), slot_pos.cpu().numpy().copy()
    for b in range(bt.B):
        n = bt.len_list[b]
        left = min(n, budget)
        for h in range(bt.Hkv):
            w = a[b, h, :n].astype(np.float64)
            w = np.where(np.isnan(w), -np.inf, w)
            nan = np.isnan(a[b, h, :n])
            pos = s[b, h, :n].astype(np.int64)
            held = (pos < sink) | (pos >= int(next_pos[b]) - recent)
            order = sorted(range(n), key=lambda i: (not held[i], nan[i] and not held[i], -w[i] if not held[i] else 0.0, i))
            kept = sorted(order[:left])
            movers = [i for i in kept if i >= left]
            holes = sorted(set(range(left)) - set(kept))
            a2, s2 = a[b, h].copy(), s[b, h].copy()
            for d, m in zip(holes, movers):
                for pool in (kp, vp):
                    pool[bt.table_list[b, d // bt.page], h, d % bt.page] = \
                        pool[bt.table_list[b, m // bt.page], h, m % bt.page]
                a2[d], s2[d] = a[b, h, m], s[b, h, m]
            a[b, h], s[b, h] = a2, s2
    return kp, vp, a, s, [min(n, budget) for n in bt.len_list]


def run_evict(bt, acc, slot_pos, next_pos, budget, recent=0, sink=0, in_place=False):
    kp, vp, a, s, lens = evict_ref(bt, acc, slot_pos, next_pos.tolist(), budget, recent, sink)
    if in_place:
        acc_o, pos_o, len_o = acc.clone(), slot_pos.clone(), bt.lens.clone()
        kernels.kv_evict(bt.kp, bt.vp, bt.table, len_o, acc_o, pos_o, next_pos, budget, recent=recent, sink=sink)
    else:
        acc_o, pos_o, len_o = torch.full_like(acc, -9.0), torch.full_like(slot_pos, -9), torch.full_like(bt.lens, -9)
        kernels.kv_evict(bt.kp, bt.vp, bt.table, bt.lens, acc, slot_pos, next_pos, budget, recent=recent, sink=sink,
                         acc_out=acc_o, slot_pos_out=pos_o, lens_out=len_o)
    kernels.device_check()
    assert len_o.tolist() == lens
    assert np.array_equal(bt.kp.view(torch.int16).cpu().numpy(), kp)
    assert np.array_equal(bt.vp.view(torch.int16).cpu().numpy(), vp)
    for b, n in enumerate(lens):
        assert np.array_equal(acc_o[b, :, :n].cpu().numpy(), a[b, :, :n], equal_nan=True)
        assert np.array_equal(pos_o[b, :, :n].cpu().numpy(), s[b, :, :n])
        if not in_place:
            assert (acc_o[b, :, n:] == -9.0).all() and (pos_o[b, :, n:] == -9).all()
        elif bt.len_list[b] > budget:  # slots above the new length keep what they held
            assert np.array_equal(acc_o[b, :, n:].cpu().numpy(), a[b, :, n:], equal_nan=True)


def weights_for(bt, kind, seed=5):
    a = torch.rand(bt.B, bt.Hkv, bt.cap, generator=gen(seed), device="cuda")
    if kind == "ties":
        a = (a * 3).floor()
    elif kind == "equal":
        a = torch.zeros_like(a)
    elif kind == "special":
        pick = torch.randint(0, 9, a.shape, generator=gen(seed + 1), device="cuda")
        for i, x in enumerate((math.nan, math.inf, -math.inf, -0.0, 0.0, -1.5, 1e-42)):
            a[pick == i] = x
    elif kind == "power":
        a = (a + 1e-3) ** -2
    return a


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "special", "power"])
@pytest.mark.parametrize("lens,budget,recent,sink,page", [
    ([1], 1, 0, 0, 16),
    ([2, 1, 0], 1, 1, 0, 16),
    ([700, 300, 512, 513], 512, 64, 4, 48),
    ([1030, 1999], 33, 0, 33, 128),
    ([65, 4097], 4096, 96, 0, 64),
    ([300], 7, 7, 0, 1),
])
def test_evict(lens, budget, recent, sink, page, kind, in_place):
    bt = Batch([0] * len(lens), lens, 4, 2, page)
    slot_pos = torch.stack([torch.stack([torch.randperm(bt.cap, generator=gen(b * 2 + h), device="cuda") for h in range(2)])
                            for b in range(bt.B)]).to(torch.int32)
    next_pos = torch.full((bt.B,), bt.cap, dtype=torch.int32, device="cuda")
    run_evict(bt, weights_for(bt, kind), slot_pos, next_pos, budget, recent, sink, in_place)


def test_evict_more_slots_than_shared_memory_holds_keys_for():
    bt = Batch([0], [60001], 1, 1, 512, extra_table=0)
    slot_pos = torch.arange(bt.cap, dtype=torch.int32, device="cuda")[None, None].contiguous()
    run_evict(bt, weights_for(bt, "ties"), slot_pos, i32([60001]), 30000, 100, 4)


def test_evict_protected_positions_win_and_bad_input_is_reported():
    bt = Batch([0, 0], [200, 100], 4, 2, 16)
    slot_pos = torch.arange(bt.cap, dtype=torch.int32, device="cuda").expand(2, 2, -1).contiguous()
    acc = torch.full((2, 2, bt.cap), math.inf, device="cuda")
    acc[:, :, :8] = 0.0
    acc[0, :, 190:200] = math.nan
    next_pos = i32([200, 100])
    pos = torch.empty_like(slot_pos)
    lens = torch.empty_like(bt.lens)
    kernels.kv_evict(bt.kp, bt.vp, bt.table, bt.lens, acc, slot_pos, next_pos, 40, recent=10, sink=8, slot_pos_out=pos,
                     lens_out=lens, acc_out=torch.empty_like(acc))
    kernels.device_check()
    for h in range(2):
        assert sorted(pos[0, h, :40].tolist()) == list(range(8)) + list(range(8, 30)) + list(range(190, 200))
    broken = bt.table.clone()
    broken[0, -2 if bt.table_list[0, -1] < 0 else -1] = -1
    kernels.kv_evict(bt.kp, bt.vp, broken, bt.lens, acc, slot_pos, next_pos, 40, recent=10, lens_out=lens)
    with pytest.raises(GqaError) as e:
        kernels.device_check()
    assert e.value.code == _lib.GQA_ERR_DEVICE_INPUT
    kernels.kv_evict(bt.kp, bt.vp, bt.table, i32([bt.cap + 1, -1]), acc, slot_pos, next_pos, bt.cap, lens_out=lens)
    with pytest.raises(GqaError):
        kernels.device_check()
    assert lens.tolist() == [bt.cap, 0]


# ------------------------------------------------------------------ refusals
def test_wrappers_refuse():
    bt = Batch([2], [20], 8, 2, 16)
    ok = dict(q=bt.q, kpages=bt.kp, vpages=bt.vp, block_table=bt.table, q_start=bt.q_start, lens=bt.lens)
    kernels.attend_chunk(**ok)
    for key, value, exc in [
        ("q", bt.q.cpu(), ValueError), ("q", bt.q.float(), TypeError), ("q", bt.q[..., ::2], ValueError),
        ("q", bt.q[:, :, :64].contiguous(), ValueError), ("q", bt.q[:, :7], GqaError),
        ("q", torch.empty(2 * 8 * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 8, D), GqaError),
        ("kpages", bt.kp.transpose(1, 2), ValueError), ("vpages", bt.vp[:-1], ValueError),
        ("block_table", bt.table.long(), TypeError), ("q_start", bt.q_start[:-1], ValueError),
        ("lens", bt.lens.long(), TypeError), ("scale", -1.0, GqaError), ("scale", math.nan, GqaError),
        ("lse", torch.empty(2, 7, device="cuda"), ValueError), ("out", bt.q.float(), TypeError),
        ("out", bt.q[:, :1].expand(2, 8, D), GqaError), ("max_q_len", -1, GqaError),
        ("workspace", torch.empty(8, dtype=torch.uint8, device="cuda"), GqaError),
    ]:
        with pytest.raises(exc):
            kernels.attend_chunk(**{**ok, key: value})
    odd = torch.zeros(4, 2, 24, D, dtype=torch.bfloat16, device="cuda")  # pages of 24 slots
    with pytest.raises(GqaError) as e:
        kernels.attend_chunk(**{**ok, "kpages": odd, "vpages": odd})
    assert e.value.code == _lib.GQA_ERR_UNSUPPORTED
    lse, acc = torch.zeros(2, 8, device="cuda"), torch.zeros(1, 2, bt.cap, device="cuda")
    args = [bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc]
    for i, value, exc in [(0, bt.q.half(), TypeError), (5, lse[:1], ValueError), (6, acc[..., 1:], ValueError),
                          (6, acc.double(), TypeError), (1, odd, ValueError)]:
        with pytest.raises(exc):
            kernels.attn_weight_sums(*args[:i], value, *args[i + 1:])
    pos, nxt = torch.zeros(1, 2, bt.cap, dtype=torch.int32, device="cuda"), i32([20])
    for kw, exc in [(dict(budget=0), GqaError), (dict(budget=4, recent=5), GqaError), (dict(budget=4, sink=-1), GqaError),
                    (dict(budget=4, workspace=torch.empty(8, dtype=torch.uint8, device="cuda")), GqaError),
                    (dict(budget=4, acc_out=acc[:, :1]), ValueError), (dict(budget=4, lens_out=bt.lens.long()), TypeError)]:
        with pytest.raises(exc):
            kernels.kv_evict(bt.kp, bt.vp, bt.table, bt.lens.clone(), acc, pos, nxt, **kw)
    k = randn(2, 2, D, seed=1)
    cos, sin = kernels.rope_table(64)
    ext = dict(k=k, v=k, kpages=bt.kp, vpages=bt.vp, block_table=bt.table, q_start=bt.q_start, lens=bt.lens, cos=cos, sin=sin)
    for key, value, exc in [("k", k[:1], ValueError), ("v", k.float(), TypeError), ("cos", None, ValueError),
                            ("sin", sin[:, :32], ValueError), ("positions", i32([1]), ValueError),
                            ("q_out", bt.q, ValueError), ("slot_pos", pos[..., 1:], ValueError)]:
        with pytest.raises(exc):
            kernels.kv_extend(**{**ext, key: value})
    with pytest.raises(GqaError):  # queries that would be written over one another
        kernels.kv_extend(**ext, q=bt.q, q_out=bt.q[:, :1].expand(2, 8, D))
    x = randn(2, 3, D, seed=2)
    for kw, exc in [(dict(positions=i32([1])), ValueError), (dict(positions=torch.zeros(2, device="cuda")), TypeError),
                    (dict(x=x.half()), TypeError), (dict(x=x[0]), ValueError), (dict(x=x[..., :32]), ValueError),
                    (dict(cos=cos.bfloat16()), TypeError), (dict(out=x[:, :1].expand(2, 3, D)), GqaError),
                    (dict(out=x.float()), TypeError)]:
        with pytest.raises(exc):
            kernels.rope_positions(**{**dict(x=x, positions=i32([1, 2]), cos=cos, sin=sin), **kw})
    kernels.device_check()


def test_no_tokens_is_no_work():
    bt = Batch([0, 0], [5, 9], 8, 2, 16)
    out = kernels.attend_chunk(bt.q, bt.kp, bt.vp, bt.table, bt.q_start, bt.lens)
    assert out.shape == (0, 8, D)
    cos, sin = kernels.rope_table(16)
    e = torch.empty(0, 2, D, dtype=torch.bfloat16, device="cuda")
    kernels.kv_extend(e, e, bt.kp, bt.vp, bt.table, bt.q_start, bt.lens, None, cos, sin)
    kernels.rope_positions(e, i32([]), cos, sin)
    # without tokens the sums pass through
    acc = torch.rand(2, 2, bt.cap, generator=gen(1), device="cuda")
    got = kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, torch.empty(0, 8, device="cuda"), acc,
                                   acc_out=torch.zeros_like(acc))
    for b, n in enumerate((5, 9)):
        assert torch.equal(got[b, :, :n], acc[b, :, :n]) and (got[b, :, n:] == 0).all()
    kernels.device_check()


# ------------------------------------------------------------------ eviction's workspace
@pytest.mark.parametrize("lens,budget", [([300, 200], 1 << 30), ([336, 40], 336), ([336, 300, 1], 335), ([40, 30], 300)])
def test_evict_workspace_of_the_rows_that_can_move(lens, budget):
    """A budget that cuts little or nothing asks for as little memory; what lies behind it stays."""
    bt = Batch([0] * len(lens), lens, 4, 2, 16, extra_table=336 // 16 - -(-max(lens) // 16))
    assert bt.cap == 336
    slot_pos = torch.arange(bt.cap, dtype=torch.int32, device="cuda").expand(bt.B, 2, -1).contiguous()
    acc = weights_for(bt, "plain")
    next_pos = i32(lens)
    need = kernels.kv_evict_workspace_bytes(bt.B, 2, budget, bt.cap)
    assert need == (0 if budget >= 336 else bt.B * 2 * (2 * min(budget, 336 - budget) + 1) * 4)
    room = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    kp, vp, a, s, left = evict_ref(bt, acc, slot_pos, lens, budget, 8, 2)
    short = bt.lens.clone()
    kernels.kv_evict(bt.kp, bt.vp, bt.table, short, acc, slot_pos, next_pos, budget, recent=8, sink=2, workspace=room[:need])
    kernels.device_check()
    assert (room[need:] == 0x5A).all() and short.tolist() == left
    assert np.array_equal(bt.kp.view(torch.int16).cpu().numpy(), kp)
    assert np.array_equal(bt.vp.view(torch.int16).cpu().numpy(), vp)
    assert np.array_equal(acc.cpu().numpy(), a) and np.array_equal(slot_pos.cpu().numpy(), s)
    run_evict(bt, acc, slot_pos, next_pos, budget, 8, 2)  # workspace from the allocator


# ------------------------------------------------------------------ the rotation under autograd
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, False), (True, True)])
def test_rope_positions_carries_its_gradient(dtype, interleaved, inverse):
    """backward is the formula's transpose, held to the rotation's own bound, and it agrees with
    differences: the rotation is linear, so <w, R(x + e) - R(x)> = <R^T w, e> up to the roundings
    of two rotations (in 32 bits, where they are small beside a step)."""
    T, H, d, rot = 21, 3, 96, 64
    cos, sin = kernels.rope_table(3000, rot, scaling="yarn", factor=4.0, original_len=1024)
    inv, m = kernels.rope_inv_freq(rot, scaling="yarn", factor=4.0, original_len=1024)
    pos = torch.randint(0, 3000, (T,), generator=gen(1), device="cuda", dtype=torch.int32)
    kw = dict(interleaved=interleaved, inverse=inverse)
    base = randn(T, H + 2, d, seed=2, dtype=dtype).requires_grad_()
    x = base[:, 1:1 + H]  # strided, as a slice of a fused projection
    y = kernels.rope_positions(x, pos, cos, sin, **kw)
    assert y.requires_grad and torch.equal(y, kernels.rope_positions(x.detach(), pos, cos, sin, **kw))
    w = randn(T, H, d, seed=3, dtype=dtype)
    g, = torch.autograd.grad(y, base, w)
    ref, mag = rope_ref(w, pos, inv, m, interleaved, not inverse)
    d_fp = 2.0 ** -22 * mag
    bound = d_fp if dtype == torch.float32 else U * (ref.abs() + d_fp) + d_fp
    assert ((g[:, 1:1 + H].double() - ref).abs() <= bound).all()
    assert (g[:, 0] == 0).all() and (g[:, 1 + H:] == 0).all()
    if dtype == torch.float32:
        e = randn(T, H, d, seed=4, dtype=dtype)
        with torch.no_grad():
            diff = kernels.rope_positions(x + e, pos, cos, sin, **kw).double() - y.double()
        lhs, rhs = (w.double() * diff).sum().item(), (g[:, 1:1 + H].double() * e.double()).sum().item()
        assert abs(lhs - rhs) <= 2.0 ** -20 * (w.double().abs() * (2 * x.double().abs() + 2 * e.double().abs())).sum().item()
    # a sum's gradient is broadcast over every dim
    ones = torch.ones(T, H, d, dtype=dtype, device="cuda")
    g, = torch.autograd.grad(kernels.rope_positions(x, pos, cos, sin, **kw).sum(), base)
    assert torch.equal(g[:, 1:1 + H], kernels.rope_positions(ones, pos, cos, sin, interleaved=interleaved, inverse=not inverse))
    # and the gradient is differentiable itself
    v = w.clone().requires_grad_()
    g, = torch.autograd.grad(kernels.rope_positions(x, pos, cos, sin, **kw), x, v, create_graph=True)
    gg, = torch.autograd.grad(g, v, w)
    assert torch.equal(gg, kernels.rope_positions(w, pos, cos, sin, **kw))
    kernels.device_check()


def test_rope_positions_refuses_gradients_that_it_does_not_carry():
    cos, sin = kernels.rope_table(8, 128)
    x, pos = randn(2, 3, D, seed=1).requires_grad_(), i32([1, 2])
    with pytest.raises(ValueError, match="out"):
        kernels.rope_positions(x, pos, cos, sin, out=torch.empty_like(x))
    with pytest.raises(ValueError, match="cos and sin"):
        kernels.rope_positions(x.detach(), pos, cos.clone().requires_grad_(), sin)
    with pytest.raises(ValueError, match="cos and sin"):
        kernels.rope_positions(x, pos, cos, sin.clone().requires_grad_())
    with torch.no_grad():  # nothing to carry
        out = torch.empty_like(x)
        assert kernels.rope_positions(x, pos, cos, sin, out=out) is out and not out.requires_grad
    kernels.device_check()


# ------------------------------------------------------------------ sizes at the ends of the ranges
def test_more_sequences_than_threads_in_a_block():
    """The split of the work takes sequences in rounds of 640: here a third begins, and a prompt lies in it."""
    B = 1500
    new = [i % 4 for i in range(B)]
    lens = [n + (7 * i) % 45 for i, n in enumerate(new)]
    new[1400], lens[1400] = 90, 400
    new[639], lens[639] = 70, 70
    bt = Batch(new, lens, 4, 1, 16, seed=41)
    lse = torch.empty(bt.T, 4, device="cuda")
    out = bt.attend(lse=lse)
    kernels.device_check()
    bt.check_attend(out, lse)
    acc = torch.rand(B, 1, bt.cap, generator=gen(8), device="cuda")
    check_weights(bt, lse, acc, kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc,
                                                         acc_out=acc.clone()))
    kernels.device_check()
    bt.kp.copy_(randn(*bt.kp.shape, seed=2))
    bt.vp.copy_(randn(*bt.vp.shape, seed=3))
    slot_pos = torch.arange(bt.cap, dtype=torch.int32, device="cuda").expand(B, 1, -1).contiguous()
    run_evict(bt, acc, slot_pos, i32(lens), 24, 4, 2)


@pytest.mark.parametrize("Hq,Hkv", [(17, 1), (128, 2), (100, 1), (256, 2)])
def test_large_groups(Hq, Hkv):
    """Up to 128 query heads share a kv head: no few-row form from 17 on, one token a tile from 65 on."""
    bt = Batch([1, 3, 0, 40], [130, 700, 20, 300], Hq, Hkv, 16, seed=43)
    for causal in (True, False):
        lse = torch.empty(bt.T, Hq, device="cuda")
        out = bt.attend(causal=causal, lse=lse)
        kernels.device_check()
        bt.check_attend(out, lse, causal)
        acc = torch.rand(4, Hkv, bt.cap, generator=gen(8), device="cuda")
        got = kernels.attn_weight_sums(bt.q, bt.kp, bt.table, bt.q_start, bt.lens, lse, acc, causal=causal, acc_out=acc.clone())
        check_weights(bt, lse, acc, got, causal)
    kernels.device_check()


@pytest.mark.parametrize("new,lens,Hq,Hkv", [([300, 1], [2300, 900], 32, 8), ([65, 40], [1025, 999], 20, 4)])
def test_attend_with_and_without_lse(new, lens, Hq, Hkv):
    """Without lse a share of the exponentials of many-row units is good to 2^-13 only, which may
    also turn a weight's rounding to bf16.  So a weight differs by at most 2 u + 2^-13 of
    itself between the calls, numerator and sum each, and the output is rounded in both."""
    bt = Batch(new, lens, Hq, Hkv, 64, seed=45)
    lse = torch.empty(bt.T, Hq, device="cuda")
    a, c = bt.attend(lse=lse).double(), bt.attend().double()
    kernels.device_check()
    G = Hq // Hkv
    for b in range(bt.B):
        n, t0 = bt.new[b], sum(bt.new[:b])
        for h in range(Hkv):
            s, _ = bt.scores(b, h, True, D ** -0.5)
            v = bt.kv(bt.vp, b, h)
            w = s.softmax(-1)
            sl = (slice(t0, t0 + n), slice(h * G, (h + 1) * G))
            bound = (2 * (2 * U + 2.0 ** -13) + 2.0 ** -12) * (w @ v.abs()) + 2 * U * (w @ v).abs()
            assert ((a[sl] - c[sl]).abs() <= bound).all()
