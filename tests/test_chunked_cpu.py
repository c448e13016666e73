"""Checks of the chunked paged-cache operators that need no GPU: argument refusals at the
C boundary (before any launch) and the scaled rotary frequencies."""
import ctypes
import math

import pytest
import torch

from llama3_8b_attention_optimize_b200 import _lib, kernels

E = _lib
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x1002)


@pytest.fixture(scope="module")
def lib():
    return _lib.load(build_if_missing=True)


def test_attend_validates_on_the_host(lib):
    def call(**kw):
        a = dict(q=FAKE, qt=1024, qh=128, kp=FAKE, vp=FAKE, table=FAKE, max_pages=4, page=16, pages=8, q_start=FAKE,
                 lens=FAKE, o=FAKE, ot=1024, oh=128, lse=None, ws=FAKE, ws_bytes=1 << 40, B=2, T=3, Hq=8, Hkv=2, d=128,
                 hint=0, scale=0.1, flags=1, **{})
        a.update(kw)
        return lib.gqa_attend_chunk_bf16(*a.values(), None)

    for bad in (dict(q=None), dict(kp=None), dict(vp=None), dict(table=None), dict(q_start=None), dict(lens=None),
                dict(o=None), dict(B=0), dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(max_pages=0), dict(page=0),
                dict(pages=0), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf), dict(flags=2), dict(hint=-1),
                dict(qt=-8), dict(oh=0), dict(ot=128), dict(oh=120)):
        assert call(**bad) == E.GQA_ERR_INVALID_ARGUMENT, bad
    for bad in (dict(d=64), dict(Hq=9), dict(page=24), dict(page=8)):
        assert call(**bad) == E.GQA_ERR_UNSUPPORTED, bad
    for bad in (dict(q=ODD), dict(kp=ODD), dict(o=ODD), dict(lens=ODD), dict(lse=ODD), dict(ws=ODD), dict(qt=1025),
                dict(qh=132)):
        assert call(**bad) == E.GQA_ERR_MISALIGNED, bad
    assert call(ws=None) == E.GQA_ERR_WORKSPACE
    assert call(ws_bytes=0) == E.GQA_ERR_WORKSPACE
    assert call(T=0, q=None) == E.GQA_OK
    assert lib.gqa_attend_chunk_workspace_size(0, 8, 2) == 0 or lib.gqa_attend_chunk_workspace_size(0, 8, 2) >= 16


def test_weight_sums_validate_on_the_host(lib):
    def call(**kw):
        a = dict(q=FAKE, qt=1024, qh=128, kp=FAKE, table=FAKE, max_pages=4, page=16, pages=8, q_start=FAKE, lens=FAKE,
                 lse=FAKE, acc=FAKE, acc_out=FAKE, ws=FAKE, ws_bytes=1 << 30, B=2, T=3, Hq=8, Hkv=2, d=128, scale=0.1,
                 flags=1)
        a.update(kw)
        return lib.gqa_attn_weight_sums_f32(*a.values(), None)

    for bad in (dict(q=None), dict(kp=None), dict(table=None), dict(q_start=None), dict(lens=None), dict(lse=None),
                dict(acc=None), dict(acc_out=None), dict(B=0), dict(T=-1), dict(scale=-1.0), dict(flags=4), dict(qh=-8)):
        assert call(**bad) == E.GQA_ERR_INVALID_ARGUMENT, bad
    for bad in (dict(d=64), dict(Hq=9), dict(page=24)):
        assert call(**bad) == E.GQA_ERR_UNSUPPORTED, bad
    for bad in (dict(q=ODD), dict(kp=ODD), dict(acc=ODD), dict(qt=4), dict(ws=ODD)):
        assert call(**bad) == E.GQA_ERR_MISALIGNED, bad
    assert call(ws=None) == E.GQA_ERR_WORKSPACE
    assert call(ws_bytes=lib.gqa_attn_weight_sums_workspace_size() - 1) == E.GQA_ERR_WORKSPACE


def test_extend_and_rope_validate_on_the_host(lib):
    def ext(**kw):
        a = dict(k=FAKE, v=FAKE, kt=256, kh=128, vt=256, vh=128, kp=FAKE, vp=FAKE, table=FAKE, max_pages=4, page=16,
                 pages=8, q_start=FAKE, lens=FAKE, pos=None, cos=FAKE, sin=FAKE, rows=8, rot=128, q=FAKE, qt=1024, qh=128,
                 qo=FAKE, ot=1024, oh=128, slot=None, B=2, T=3, Hq=8, Hkv=2, d=128, flags=0)
        a.update(kw)
        return lib.gqa_kv_extend_bf16(*a.values(), None)

    for bad in (dict(k=None), dict(v=None), dict(kp=None), dict(vp=None), dict(table=None), dict(q_start=None),
                dict(lens=None), dict(cos=None), dict(rows=0), dict(rot=130), dict(rot=3), dict(rot=-2), dict(qo=None),
                dict(q=None), dict(Hq=0), dict(B=0), dict(T=-1), dict(page=0), dict(flags=16), dict(kt=-1), dict(oh=64),
                dict(ot=512)):
        assert ext(**bad) == E.GQA_ERR_INVALID_ARGUMENT, bad
    assert ext(d=64) == E.GQA_ERR_UNSUPPORTED
    for bad in (dict(kp=ODD), dict(lens=ODD), dict(cos=ODD), dict(k=ctypes.c_void_p(0x1001))):
        assert ext(**bad) == E.GQA_ERR_MISALIGNED, bad
    assert ext(T=0, k=None) == E.GQA_OK

    def rope(fn, **kw):
        a = dict(x=FAKE, y=FAKE, pos=FAKE, cos=FAKE, sin=FAKE, T=3, H=2, d=128, rot=64, rows=8, xt=256, xh=128, yt=256,
                 yh=128, flags=0)
        a.update(kw)
        return fn(*a.values(), None)

    for fn in (lib.gqa_rope_positions_bf16, lib.gqa_rope_positions_f32):
        for bad in (dict(x=None), dict(y=None), dict(pos=None), dict(cos=None), dict(T=-1), dict(H=0), dict(rot=0),
                    dict(rot=63), dict(rot=130), dict(rows=0), dict(flags=1), dict(xt=-1), dict(yh=0), dict(yt=100)):
            assert rope(fn, **bad) == E.GQA_ERR_INVALID_ARGUMENT, bad
        assert rope(fn, d=1024, xt=2048, xh=1024, yt=2048, yh=1024) == E.GQA_ERR_UNSUPPORTED
        assert rope(fn, y=ctypes.c_void_p(0x1001)) == E.GQA_ERR_MISALIGNED
        assert rope(fn, T=0, x=None) == E.GQA_OK
    for bad in ((None, FAKE, FAKE, 4, 64, 0, 1.0), (FAKE, FAKE, FAKE, 0, 64, 0, 1.0), (FAKE, FAKE, FAKE, 4, 64, -1, 1.0),
                (FAKE, FAKE, FAKE, 4, 64, 0, 0.0), (FAKE, FAKE, FAKE, 4, 64, 0, math.nan)):
        assert lib.gqa_rope_table_f32(*bad, None) == E.GQA_ERR_INVALID_ARGUMENT


def test_evict_validates_on_the_host(lib):
    assert lib.gqa_kv_evict_workspace_size(2, 8, 100) == 2 * 8 * 201 * 4
    assert lib.gqa_kv_evict_workspace_size(0, 8, 100) == 0

    def call(**kw):
        a = dict(kp=FAKE, vp=FAKE, table=FAKE, max_pages=4, page=16, pages=8, lens=FAKE, lens_out=FAKE, acc=FAKE,
                 acc_out=FAKE, pos=FAKE, pos_out=FAKE, nxt=FAKE, ws=FAKE, ws_bytes=1 << 30, B=2, Hkv=2, d=128, budget=32,
                 recent=4, sink=4)
        a.update(kw)
        return lib.gqa_kv_evict_bf16(*a.values(), None)

    for bad in (dict(kp=None), dict(vp=None), dict(table=None), dict(lens=None), dict(lens_out=None), dict(acc=None),
                dict(acc_out=None), dict(pos=None), dict(pos_out=None), dict(nxt=None), dict(budget=0), dict(recent=-1),
                dict(sink=-1), dict(recent=30), dict(B=0), dict(page=0)):
        assert call(**bad) == E.GQA_ERR_INVALID_ARGUMENT, bad
    assert call(d=64) == E.GQA_ERR_UNSUPPORTED
    assert call(max_pages=1 << 20, page=16) == E.GQA_ERR_UNSUPPORTED
    assert call(kp=ODD) == E.GQA_ERR_MISALIGNED
    assert call(acc=ODD) == E.GQA_ERR_MISALIGNED
    assert call(ws=None) == E.GQA_ERR_WORKSPACE
    assert call(ws_bytes=16) == E.GQA_ERR_WORKSPACE


def test_packed_calls_match_their_declarations(lib):
    """Packed argument counts are those of the ctypes signatures without scale and stream;
    other counts, entries and integers too wide for their argument are refused."""
    import struct
    for name, (entry, n) in E.PACKED.items():
        args = E.SIGNATURES[name][1]
        assert n == sum(1 for a in args if a is not ctypes.c_float) - 1
        for count in (n - 1, n + 1, 0):
            assert lib.gqa_packed_call(entry, struct.pack(f"{n}q", *[0] * n), count, 0.1, None) == E.GQA_ERR_INVALID_ARGUMENT
        assert lib.gqa_packed_call(entry, struct.pack(f"{n}q", *[0] * n), n, 0.1, None) == E.GQA_ERR_INVALID_ARGUMENT
    entry, n = E.PACKED["gqa_rope_positions_bf16"]
    good = [0x1000] * 5 + [0, 2, 128, 64, 8, 256, 128, 256, 128, 0]  # T = 0: nothing to do
    assert lib.gqa_packed_call(entry, struct.pack(f"{n}q", *good), n, 0.0, None) == E.GQA_OK
    good[5] = 1 << 32
    assert lib.gqa_packed_call(entry, struct.pack(f"{n}q", *good), n, 0.0, None) == E.GQA_ERR_INVALID_ARGUMENT
    assert lib.gqa_packed_call(99, struct.pack("1q", 0), 1, 0.0, None) == E.GQA_ERR_INVALID_ARGUMENT
    assert lib.gqa_packed_call(0, None, 15, 0.0, None) == E.GQA_ERR_INVALID_ARGUMENT


def test_scaled_frequencies():
    base, m = kernels.rope_inv_freq(128)
    assert m == 1.0 and base[0] == 1.0 and torch.allclose(base, 500000.0 ** (-torch.arange(64).double() / 64))
    lin, m = kernels.rope_inv_freq(128, scaling="linear", factor=4.0)
    assert m == 1.0 and torch.equal(lin, base / 4.0)
    # blended by wavelength: short ones kept, long ones divided, in between monotone
    l3, m = kernels.rope_inv_freq(128, scaling="llama3", factor=8.0, original_len=8192)
    wave = 2 * math.pi / base
    assert m == 1.0
    assert torch.equal(l3[wave < 8192 / 4.0], base[wave < 8192 / 4.0])
    assert torch.equal(l3[wave > 8192], base[wave > 8192] / 8.0)
    mid = (wave >= 8192 / 4.0) & (wave <= 8192)
    assert mid.any() and (l3[mid] < base[mid]).all() and (l3[mid] > base[mid] / 8.0).all()
    for i in mid.nonzero()[:, 0].tolist():
        smooth = (8192 / wave[i].item() - 1.0) / (4.0 - 1.0)
        assert math.isclose(l3[i].item(), (1 - smooth) * base[i].item() / 8.0 + smooth * base[i].item(), rel_tol=1e-12)
    ya, m = kernels.rope_inv_freq(128, theta=10000.0, scaling="yarn", factor=16.0, original_len=4096)
    b = kernels.rope_inv_freq(128, theta=10000.0)[0]
    assert math.isclose(m, 0.1 * math.log(16.0) + 1.0)
    turns = 4096 * b / (2 * math.pi)
    assert torch.equal(ya[turns > 40], b[turns > 40]) and torch.allclose(ya[turns < 0.7], b[turns < 0.7] / 16.0, rtol=1e-12)
    assert ((ya / b).diff() <= 1e-12).all()
    for kw in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=8, scaling="none", factor=0.5), dict(rot_dim=8, theta=1.0),
               dict(rot_dim=8, scaling="other"), dict(rot_dim=8, scaling="llama3", low_freq=4.0, high_freq=1.0),
               dict(rot_dim=8, scaling="yarn", beta_fast=1.0, beta_slow=32.0)):
        with pytest.raises(ValueError):
            kernels.rope_inv_freq(**kw)


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    c = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.rope_positions(x, i, c, c)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.attend_chunk(x, x, x, i, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.attn_weight_sums(x, x, i, i, i, c, c)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.kv_extend(x, x, x, x, i, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.kv_evict(x, x, i, i, c, i, i, 4)
    with pytest.raises(TypeError):
        kernels.rope_positions([1.0], i, c, c)


def test_package_imports_under_a_torch_without_cuda():
    """Such a torch has no _cuda_ names in torch._C; what needs no GPU works there."""
    import subprocess
    import sys
    code = ("import torch\n"
            "for name in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    delattr(torch._C, name)\n"
            "from llama3_8b_attention_optimize_b200 import kernels, golden_model, cpu_baseline\n"
            "print(kernels.rope_inv_freq(4)[0].tolist()[0])\n")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == "1.0", run.stderr


def test_evict_workspace_goes_by_the_rows_that_can_move(lib):
    """Of a sequence's slots at most min(budget, capacity - budget) change their place."""
    assert kernels.kv_evict_workspace_bytes(32, 8, 1 << 30, 32768) == 0  # nothing is ever cut
    assert kernels.kv_evict_workspace_bytes(32, 8, 32768, 32768) == 0
    assert kernels.kv_evict_workspace_bytes(2, 8, 4096, 4097) == lib.gqa_kv_evict_workspace_size(2, 8, 1)
    assert kernels.kv_evict_workspace_bytes(2, 8, 100, 32768) == lib.gqa_kv_evict_workspace_size(2, 8, 100)
    assert kernels.kv_evict_workspace_bytes(2, 8, 100) == lib.gqa_kv_evict_workspace_size(2, 8, 100)


def test_attend_workspace_holds_two_parts_a_cta(lib):
    """148 CTAs leave at most two parts of a unit, each 128 values, a maximum and two sums a row, and
    a descriptor of 32 bytes; without tokens nothing is needed."""
    assert lib.gqa_attend_chunk_workspace_size(0, 8, 2) == 0
    for T, Hq, Hkv, rows in [(1, 8, 2, 4), (32, 8, 2, 128), (33, 8, 2, 256), (5000, 32, 8, 256), (1, 128, 1, 128), (2, 100, 1, 256)]:
        sums = -(-(2 * 148 * 3 * rows * 4) // 16) * 16
        assert lib.gqa_attend_chunk_workspace_size(T, Hq, Hkv) == 2 * 148 * 128 * rows * 4 + sums + 148 * 32
