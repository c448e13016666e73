"""Torch-facing wrappers over the C ABI (one function per entry point).

All tensors are CUDA bf16, contiguous; calls are enqueued on the current torch
stream.  Shapes follow the reference's golden model: per-head [H][S][d], with an
optional leading batch axis.  Raises ``GqaError`` on any non-zero status.
"""
from __future__ import annotations

import math
import struct

import torch

from . import _lib
from ._lib import (GQA_FLAG_CAUSAL, GQA_FLAG_INTERLEAVED, GQA_FLAG_INVERSE, GQA_FLAG_ROPE_K, GQA_FLAG_ROPE_Q,
                   GQA_GEMM_OUT_F32, GqaError, check)

ROPE_THETA = 500000.0
HEAD_DIM = 128


def default_scale(head_dim: int = HEAD_DIM) -> float:
    """fl32(1/sqrt(d)), the golden's ``scale`` (llama3_attention_golden_model.py:175)."""
    return float(torch.tensor(1.0 / math.sqrt(head_dim), dtype=torch.float32))


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


def _need(t: torch.Tensor, name: str, dtype=torch.bfloat16) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the kernels have no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def rope_cache(seq_len: int, head_dim: int = HEAD_DIM, theta: float = ROPE_THETA, pos0: int = 0,
               device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) bf16 [seq_len][head_dim] on the device (golden build_rope_cache :124-130)."""
    device = torch.device(device or "cuda")
    cos = torch.empty(seq_len, head_dim, dtype=torch.bfloat16, device=device)
    sin = torch.empty_like(cos)
    check(_lib.load().gqa_rope_cache_bf16(_ptr(cos), _ptr(sin), seq_len, head_dim, pos0, float(theta),
                                          _stream(device)), "gqa_rope_cache_bf16")
    return cos, sin


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos0: int = 0,
         out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16(x*cos + rotate_half(x)*sin) for x [..., S, d] (golden apply_rope :133-139)."""
    _need(x, "x")
    _need(cos, "cos")
    _need(sin, "sin")
    S, d = x.shape[-2], x.shape[-1]
    if cos.shape[-1] != d or cos.shape[0] < pos0 + S:
        raise ValueError("rope table too short or wrong width")
    out = torch.empty_like(x) if out is None else out
    _need(out, "out")
    heads = x.numel() // (S * d)
    check(_lib.load().gqa_rope_bf16(_ptr(x), _ptr(out), _ptr(cos), _ptr(sin), heads, S, d, pos0, _stream(x.device)),
          "gqa_rope_bf16")
    return out


def _bhsd(x: torch.Tensor, name: str) -> torch.Tensor:
    if x.dim() == 3:
        return x.unsqueeze(0)
    if x.dim() != 4:
        raise ValueError(f"{name} must be [H,S,d] or [B,H,S,d]")
    return x


def scores(q: torch.Tensor, k: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    """bf16(q k^T * scale) [B,Hq,S,S] (golden scores_before_mask :175-176)."""
    _need(q, "q")
    _need(k, "k")
    q4, k4 = _bhsd(q, "q"), _bhsd(k, "k")
    B, Hq, S, d = q4.shape
    Hkv = k4.shape[1]
    out = torch.empty(B, Hq, S, S, dtype=torch.bfloat16, device=q.device)
    check(_lib.load().gqa_scores_bf16(_ptr(q4), _ptr(k4), _ptr(out), B, Hq, Hkv, S, d,
                                      default_scale(d) if scale is None else float(scale), _stream(q.device)),
          "gqa_scores_bf16")
    return out if q.dim() == 4 else out[0]


def mask(s: torch.Tensor, causal: bool = True) -> torch.Tensor:
    """bf16(s + triu(-inf, 1)) (golden scores_after_mask :180-181)."""
    _need(s, "scores")
    S = s.shape[-1]
    out = torch.empty_like(s)
    check(_lib.load().gqa_mask_bf16(_ptr(s), _ptr(out), s.numel() // (S * S), S, int(causal), _stream(s.device)),
          "gqa_mask_bf16")
    return out


def attention_mask_words(raw: torch.Tensor, q_heads: int, seq_len: int, causal: bool = True,
                         mask_value: int = _lib.GQA_MASK_NEG_INF_BF16) -> torch.Tensor:
    """Raw-word mask of the HLS kernel (attention_mask.cpp:3-58) on int16/bf16 words."""
    if raw.dtype not in (torch.int16, torch.bfloat16, torch.uint16):
        raise TypeError("raw must hold 16-bit words")
    if not raw.is_cuda or not raw.is_contiguous():
        raise ValueError("raw must be a contiguous CUDA tensor")
    out = torch.empty_like(raw)
    check(_lib.load().gqa_attention_mask_bf16(_ptr(raw), _ptr(out), q_heads, seq_len, int(causal), mask_value,
                                              _stream(raw.device)), "gqa_attention_mask_bf16")
    return out


def softmax(s: torch.Tensor) -> torch.Tensor:
    """bf16(softmax(s, -1)) (golden softmax_weights :185)."""
    _need(s, "scores")
    out = torch.empty_like(s)
    cols = s.shape[-1]
    check(_lib.load().gqa_softmax_bf16(_ptr(s), _ptr(out), s.numel() // cols, cols, _stream(s.device)),
          "gqa_softmax_bf16")
    return out


def pv(p: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """bf16(p v) with fp32 accumulation (golden attn_out_per_head :189)."""
    _need(p, "probs")
    _need(v, "v")
    p4, v4 = _bhsd(p, "p"), _bhsd(v, "v")
    B, Hq, S, _ = p4.shape
    Hkv, d = v4.shape[1], v4.shape[3]
    out = torch.empty(B, Hq, S, d, dtype=torch.bfloat16, device=p.device)
    check(_lib.load().gqa_pv_bf16(_ptr(p4), _ptr(v4), _ptr(out), B, Hq, Hkv, S, d, _stream(p.device)), "gqa_pv_bf16")
    return out if p.dim() == 4 else out[0]


def prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor | None = None,
            sin: torch.Tensor | None = None, *, causal: bool = True, rope_q: bool = False, rope_k: bool = False,
            scale: float | None = None, kv_heads: tuple[int, int] | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """Fused GQA attention core (tcgen05): O = softmax(mask(rope(Q) rope(K)^T * scale)) V.

    q [B,Hq,S,128], k/v [B,Hkv,S,128] (or without B); rope_q/rope_k rotate in the
    kernel with the (cos, sin) tables of ``rope_cache``.  ``kv_heads=(begin, count)``
    restricts the work to one KV-head shard; other heads of ``out`` are untouched.
    """
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, n)
    q4, k4, v4 = _bhsd(q, "q"), _bhsd(k, "k"), _bhsd(v, "v")
    B, Hq, S, d = q4.shape
    Hkv = k4.shape[1]
    if k4.shape != (B, Hkv, S, d) or v4.shape != k4.shape:
        raise ValueError("k and v must be [B,Hkv,S,d] matching q")
    flags = (GQA_FLAG_CAUSAL if causal else 0) | (GQA_FLAG_ROPE_Q if rope_q else 0) | (GQA_FLAG_ROPE_K if rope_k else 0)
    if (rope_q or rope_k):
        if cos is None or sin is None:
            raise ValueError("rope_q/rope_k need cos and sin tables")
        _need(cos, "cos")
        _need(sin, "sin")
        if cos.shape[0] < S or cos.shape[1] != d:
            raise ValueError("rope table shorter than the sequence")
    if out is None:
        out = torch.empty_like(q4)
    _need(out, "out")
    kb, kc = (0, Hkv) if kv_heads is None else kv_heads
    check(_lib.load().gqa_prefill_bf16(_ptr(q4), _ptr(k4), _ptr(v4), _ptr(out),
                                       _ptr(cos) if cos is not None else None, _ptr(sin) if sin is not None else None,
                                       B, S, Hq, Hkv, d, kb, kc, default_scale(d) if scale is None else float(scale),
                                       flags, _stream(q.device)), "gqa_prefill_bf16")
    return out if q.dim() == 4 else out[0]


def decode_workspace_bytes(B: int, Hq: int, max_len: int, split_len: int = 0) -> int:
    return int(_lib.load().gqa_decode_workspace_size(B, Hq, max_len, split_len))


def decode(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, lens: torch.Tensor, *,
           q_pos: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None, split_len: int = 0, scale: float | None = None,
           kv_heads: tuple[int, int] | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Split-KV decode: q [B,Hq,128] against kcache/vcache [B,Hkv,Lmax,128]; lens int32 [B].

    With ``q_pos`` (int32 [B]) and (cos, sin), q is rotated at q_pos[b] in the kernel.
    """
    for t, n in ((q, "q"), (kcache, "kcache"), (vcache, "vcache")):
        _need(t, n)
    _need(lens, "lens", torch.int32)
    B, Hq, d = q.shape
    Hkv, Lmax = kcache.shape[1], kcache.shape[2]
    if kcache.shape != (B, Hkv, Lmax, d) or vcache.shape != kcache.shape or lens.shape != (B,):
        raise ValueError("bad decode shapes")
    flags = 0
    if q_pos is not None:
        _need(q_pos, "q_pos", torch.int32)
        _need(cos, "cos")
        _need(sin, "sin")
        if cos.shape[0] < Lmax + 1 or sin.shape[0] < Lmax + 1:
            raise ValueError("decode rope tables need max_len + 1 rows")
        flags |= GQA_FLAG_ROPE_Q
    need = decode_workspace_bytes(B, Hq, Lmax, split_len)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    out = torch.empty_like(q) if out is None else out
    kb, kc = (0, Hkv) if kv_heads is None else kv_heads
    check(_lib.load().gqa_decode_bf16(_ptr(q), _ptr(kcache), _ptr(vcache), _ptr(lens),
                                      _ptr(q_pos) if q_pos is not None else None,
                                      _ptr(cos) if cos is not None else None, _ptr(sin) if sin is not None else None,
                                      _ptr(out), _ptr(workspace), workspace.numel() * workspace.element_size(),
                                      B, Lmax, Hq, Hkv, d, kb, kc, split_len,
                                      default_scale(d) if scale is None else float(scale), flags, _stream(q.device)),
          "gqa_decode_bf16")
    return out


def kv_append(k_new: torch.Tensor, v_new: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor,
              lens: torch.Tensor, *, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
              block_table: torch.Tensor | None = None, lens_out: torch.Tensor | None = None) -> None:
    """Write k_new/v_new [B,Hkv,n,128] at positions lens[b] + i of the cache, K rotated
    there when (cos, sin) are given.  Contiguous cache [B,Hkv,Lmax,128], or (with
    ``block_table`` int32 [B,max_pages]) page pools [num_pages,Hkv,page_size,128].
    ``lens_out`` (may be ``lens``) receives lens + n after the writes."""
    for t, n in ((k_new, "k_new"), (v_new, "v_new"), (kcache, "kcache"), (vcache, "vcache")):
        _need(t, n)
    _need(lens, "lens", torch.int32)
    B, Hkv, n, d = k_new.shape
    if v_new.shape != k_new.shape or vcache.shape != kcache.shape or lens.shape != (B,):
        raise ValueError("bad kv_append shapes")
    flags = 0
    if cos is not None or sin is not None:
        _need(cos, "cos")
        _need(sin, "sin")
        flags |= GQA_FLAG_ROPE_K
    if block_table is not None:
        _need(block_table, "block_table", torch.int32)
        num_pages, _, page_size, _ = kcache.shape
        max_pages, max_len = block_table.shape[1], 0
        if block_table.shape[0] != B or kcache.shape[1] != Hkv:
            raise ValueError("bad paged kv_append shapes")
    else:
        if kcache.shape[:2] != (B, Hkv):
            raise ValueError("bad kv_append cache shape")
        num_pages = page_size = max_pages = 0
        max_len = kcache.shape[2]
    if lens_out is not None:
        _need(lens_out, "lens_out", torch.int32)
    capacity = max_pages * page_size if block_table is not None else max_len
    if flags and (cos.shape[0] < capacity or sin.shape[0] < capacity):
        raise ValueError("kv_append rope tables need one row per cache position")
    check(_lib.load().gqa_kv_append_bf16(_ptr(k_new), _ptr(v_new), _ptr(kcache), _ptr(vcache),
                                         _ptr(block_table) if block_table is not None else None, max_pages, page_size,
                                         num_pages, _ptr(lens), _ptr(lens_out) if lens_out is not None else None,
                                         _ptr(cos) if cos is not None else None, _ptr(sin) if sin is not None else None,
                                         B, Hkv, n, d, max_len, flags, _stream(k_new.device)), "gqa_kv_append_bf16")


def decode_paged(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor,
                 lens: torch.Tensor, *, q_pos: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, workspace: torch.Tensor | None = None, split_len: int = 0,
                 scale: float | None = None, kv_heads: tuple[int, int] | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Split-KV decode over page pools kpages/vpages [num_pages,Hkv,page_size,128] with
    block_table int32 [B,max_pages] (page_size a multiple of 128)."""
    for t, n in ((q, "q"), (kpages, "kpages"), (vpages, "vpages")):
        _need(t, n)
    _need(lens, "lens", torch.int32)
    _need(block_table, "block_table", torch.int32)
    B, Hq, d = q.shape
    num_pages, Hkv, page_size, _ = kpages.shape
    max_pages = block_table.shape[1]
    if vpages.shape != kpages.shape or block_table.shape[0] != B or lens.shape != (B,):
        raise ValueError("bad paged decode shapes")
    capacity = max_pages * page_size
    flags = 0
    if q_pos is not None:
        _need(q_pos, "q_pos", torch.int32)
        _need(cos, "cos")
        _need(sin, "sin")
        if cos.shape[0] < capacity + 1 or sin.shape[0] < capacity + 1:
            raise ValueError("decode rope tables need capacity + 1 rows")
        flags |= GQA_FLAG_ROPE_Q
    need = decode_workspace_bytes(B, Hq, capacity, split_len)
    if workspace is None:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    out = torch.empty_like(q) if out is None else out
    kb, kc = (0, Hkv) if kv_heads is None else kv_heads
    check(_lib.load().gqa_decode_paged_bf16(_ptr(q), _ptr(kpages), _ptr(vpages), _ptr(block_table), max_pages,
                                            page_size, num_pages, _ptr(lens),
                                            _ptr(q_pos) if q_pos is not None else None,
                                            _ptr(cos) if cos is not None else None,
                                            _ptr(sin) if sin is not None else None, _ptr(out), _ptr(workspace),
                                            workspace.numel() * workspace.element_size(), B, Hq, Hkv, d, kb, kc,
                                            split_len, default_scale(d) if scale is None else float(scale), flags,
                                            _stream(q.device)), "gqa_decode_paged_bf16")
    return out


# ------------------------------------------------------------------ serving a paged cache chunk by chunk
# A step brings a ragged batch of new tokens: sequence b owns tokens
# [q_start[b], q_start[b + 1]) and lens[b] counts its cached slots with those tokens
# included, so its token i of n sits in slot lens[b] - n + i.  For serving: of these calls only
# rope_positions takes part in autograd, the others' results carry no gradient.

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_SCALE = default_scale()
# (device index) -> cudaStream_t, without a Stream object; None in a torch built without CUDA
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _rows3(t: torch.Tensor, name: str, dtype=torch.bfloat16) -> None:
    """A CUDA [T, H, d] tensor whose last dim is contiguous; any token and head strides."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the kernels have no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 3 or (t.stride(2) != 1 and t.shape[2] > 1):
        raise ValueError(f"{name} must be [T, H, d] with a contiguous last dim")


def _no_broadcast(t: torch.Tensor) -> torch.Tensor:
    """t itself, or a copy where tokens or heads share memory (TMA reads along strides above zero)."""
    T, H, _ = t.shape
    return t.contiguous() if (T > 1 and t.stride(0) == 0) or (H > 1 and t.stride(1) == 0) else t


def _check(dev: int, rows: tuple, flat: tuple) -> None:
    """Checks of one call's tensors: rows = (tensor or None, name, dtype) of [T, H, d] tensors with
    a contiguous last dim, flat = the same of contiguous ones, all on device index `dev`.  A
    call's checks cost the host as much as a short kernel takes, so the usual case is one
    pass of cheap tests; what fails one is looked at again for its message."""
    for t, name, dtype in rows:
        if t is not None and not (t.__class__ is torch.Tensor and t.dtype is dtype and t.get_device() == dev and
                                  t.dim() == 3 and t.stride(2) == 1):
            _rows3(t, name, dtype)
            if t.get_device() != dev:
                raise ValueError("all tensors must be on one device")
    for t, name, dtype in flat:
        if t is not None and not (t.__class__ is torch.Tensor and t.dtype is dtype and t.get_device() == dev and
                                  t.is_contiguous()):
            _need(t, name, dtype)
            if t.get_device() != dev:
                raise ValueError("all tensors must be on one device")


def _index(t: torch.Tensor, name: str) -> int:
    """The CUDA device index of a call's first tensor."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the kernels have no CPU path)")
    return t.get_device()


_packers = {name: (entry, n, struct.Struct(f"{n}q").pack) for name, (entry, n) in _lib.PACKED.items()}


def _call(dev: int, name: str, scale: float, *args: int) -> None:
    """Enqueue one entry point of ``gqa_packed_call`` on the current torch stream of device
    index `dev` (ctypes converts some 30 arguments in 4 us, one packed array in 1)."""
    entry, n, pack = _packers[name]
    fn = _lib.load().gqa_packed_call
    if torch._C._cuda_getDevice() == dev:
        rc = fn(entry, pack(*args), n, scale, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(entry, pack(*args), n, scale, _raw_stream(dev))
    if rc != 0:
        check(rc, name)


def _workspace(workspace: torch.Tensor | None, need: int, dev: int) -> torch.Tensor:
    """The caller's workspace, or one of `need` bytes from torch's allocator (whose streams it follows)."""
    if workspace is None:
        return torch.empty(max(need, 16), dtype=torch.uint8, device=_devices[dev])
    if not isinstance(workspace, torch.Tensor) or workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on the same device")
    return workspace


class _Devices(dict):
    def __missing__(self, index: int) -> torch.device:
        return self.setdefault(index, torch.device("cuda", index))


_devices = _Devices()


def rope_inv_freq(rot_dim: int, theta: float = ROPE_THETA, *, scaling: str = "none", factor: float = 1.0,
                  original_len: int = 8192, low_freq: float = 1.0, high_freq: float = 4.0, beta_fast: float = 32.0,
                  beta_slow: float = 1.0) -> tuple[torch.Tensor, float]:
    """(inv_freq float64 [rot_dim/2], mscale): theta^(-2i/rot_dim), stretched for contexts
    ``factor`` times longer than ``original_len``.

    none     as they are
    linear   every frequency divided by factor (positions interpolated)
    llama3   wavelengths above original_len/low_freq divided by factor, below
             original_len/high_freq kept, in between a linear blend in original_len/wavelength
    yarn     dims that turn at least beta_fast times within original_len kept, at most
             beta_slow times divided by factor, a linear ramp over the dims in between;
             mscale = 0.1 ln(factor) + 1 on cos and sin
    """
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even and positive")
    if not theta > 1.0 or not factor >= 1.0 or original_len <= 0:
        raise ValueError("theta > 1, factor >= 1 and original_len > 0 are needed")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    inv = theta ** (-i / rot_dim)
    if scaling == "none":
        return inv, 1.0
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "llama3":
        if not 0 < low_freq < high_freq:
            raise ValueError("0 < low_freq < high_freq is needed")
        turns = original_len * inv / (2 * math.pi)  # original_len / wavelength
        keep = ((turns - low_freq) / (high_freq - low_freq)).clamp(0.0, 1.0)
        return inv * keep + inv / factor * (1.0 - keep), 1.0
    if scaling == "yarn":
        if not 0 < beta_slow < beta_fast:
            raise ValueError("0 < beta_slow < beta_fast is needed")
        def dim_of(turns: float) -> float:  # the dim pair that turns so often within original_len
            return rot_dim * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo = max(math.floor(dim_of(beta_fast)), 0)
        hi = min(math.ceil(dim_of(beta_slow)), rot_dim - 1)
        stretch = ((torch.arange(rot_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        return inv / factor * stretch + inv * (1.0 - stretch), 0.1 * math.log(factor) + 1.0
    raise ValueError("scaling must be none, linear, llama3 or yarn")


def rope_table(rows: int, rot_dim: int = HEAD_DIM, theta: float = ROPE_THETA, pos0: int = 0, device=None,
               **scaling) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) float32 [rows][rot_dim/2] of positions pos0 .. pos0 + rows - 1 for
    ``rope_positions`` and ``kv_extend``, from 64-bit angles; ``scaling`` as in ``rope_inv_freq``."""
    inv, mscale = rope_inv_freq(rot_dim, theta, **scaling)
    device = torch.device(device or "cuda")
    inv = inv.to(device)
    cos = torch.empty(rows, rot_dim // 2, dtype=torch.float32, device=device)
    sin = torch.empty_like(cos)
    with torch.cuda.device(cos.device):
        check(_lib.load().gqa_rope_table_f32(_ptr(inv), _ptr(cos), _ptr(sin), rows, rot_dim // 2, pos0, mscale,
                                             _stream(cos.device)), "gqa_rope_table_f32")
    return cos, sin


def rope_positions(x: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                   interleaved: bool = False, inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, H, d] (bf16 or float32, any token and head strides) rotated at positions[t]
    (int32 [T]) over its first 2 * cos.shape[1] dims; the others pass through.

    cos, sin: ``rope_table``.  Pairs are (i, i + rot/2), or (2i, 2i + 1) when ``interleaved``.
    ``inverse`` rotates backwards, which is the gradient's way through this operator: where x
    requires a gradient autograd takes it, in x's type (the tables get none, and ``out``
    carries none: both are refused).  ``out`` may be x."""
    dev = _index(x, "x")
    if x.dtype is not _BF16 and x.dtype is not _F32:
        raise TypeError(f"x must be bfloat16 or float32, got {x.dtype}")
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out carries no gradient: leave it away, or pass x detached")
        return _RopePositions.apply(x, positions, cos, sin, interleaved, inverse)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    _check(dev, ((x, "x", x.dtype), (out, "out", x.dtype)),
           ((positions, "positions", _I32), (cos, "cos", _F32), (sin, "sin", _F32)))
    if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise ValueError("cos and sin get no gradient: pass them detached")
    T, H, d = x.shape
    if positions.shape != (T,):
        raise ValueError("positions must be [T]")
    if cos.dim() != 2 or sin.shape != cos.shape or 2 * cos.shape[1] > d:
        raise ValueError("cos and sin must be [rows, rot/2] with rot <= d")
    if out.shape != x.shape:
        raise ValueError("out must have x's shape")
    rows, half = cos.shape
    _call(dev, "gqa_rope_positions_bf16" if x.dtype is _BF16 else "gqa_rope_positions_f32", 0.0, x.data_ptr(), out.data_ptr(),
          positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), T, H, d, 2 * half, rows, x.stride(0), x.stride(1),
          out.stride(0), out.stride(1), (GQA_FLAG_INTERLEAVED if interleaved else 0) | (GQA_FLAG_INVERSE if inverse else 0))
    return out


class _RopePositions(torch.autograd.Function):
    """``rope_positions`` of an x that requires a gradient: the rotation is linear in x, and its
    transpose is the rotation backwards (times the same scale of the tables)."""

    @staticmethod
    def forward(ctx, x, positions, cos, sin, interleaved, inverse):
        if any(ctx.needs_input_grad[1:4]):
            raise ValueError("cos and sin get no gradient: pass them detached")
        ctx.save_for_backward(positions, cos, sin)
        ctx.interleaved, ctx.inverse = interleaved, inverse
        return rope_positions(x, positions, cos, sin, interleaved=interleaved, inverse=inverse)

    @staticmethod
    def backward(ctx, grad):
        positions, cos, sin = ctx.saved_tensors
        grad = grad if grad.stride(-1) == 1 else grad.contiguous()  # a broadcast one, as a sum's
        g = rope_positions(grad, positions, cos, sin, interleaved=ctx.interleaved, inverse=not ctx.inverse)
        return g, None, None, None, None, None


def _paged(kpages: torch.Tensor, vpages: torch.Tensor | None, block_table: torch.Tensor, q_start: torch.Tensor | None,
           lens: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(B, max_pages, page_size, num_pages, Hkv) of page pools and tables with fitting shapes."""
    shape = kpages.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM or (vpages is not None and vpages.shape != shape):
        raise ValueError("kpages and vpages must be [num_pages, Hkv, page_size, 128]")
    num_pages, Hkv, page_size, _ = shape
    if block_table.dim() != 2 or lens.shape != (block_table.shape[0],):
        raise ValueError("block_table must be [B, max_pages] and lens [B]")
    B, max_pages = block_table.shape
    if q_start is not None and q_start.shape != (B + 1,):
        raise ValueError("q_start must be [B + 1]")
    return B, max_pages, page_size, num_pages, Hkv


def kv_extend(k: torch.Tensor, v: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor,
              q_start: torch.Tensor, lens: torch.Tensor, positions: torch.Tensor | None = None,
              cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *, q: torch.Tensor | None = None,
              q_out: torch.Tensor | None = None, interleaved: bool = False,
              slot_pos: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write the new tokens' k and v [T, Hkv, 128] into their slots of the page pools, k
    rotated at positions[t] (int32 [T]; None: at its slot) when the ``rope_table`` tables
    are given.  With ``q`` [T, Hq, 128], rotates the queries too and returns them
    (``q_out``, which may be q).  ``slot_pos`` (int32 [B, Hkv, capacity]) receives the
    position held by each slot written, for ``kv_evict``."""
    dev = _index(k, "k")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=_BF16, device=k.device)
    elif q is None and q_out is not None:
        raise ValueError("q_out needs q")
    _check(dev, ((k, "k", _BF16), (v, "v", _BF16), (q, "q", _BF16), (q_out, "q_out", _BF16)),
           ((kpages, "kpages", _BF16), (vpages, "vpages", _BF16), (block_table, "block_table", _I32),
            (q_start, "q_start", _I32), (lens, "lens", _I32), (positions, "positions", _I32), (cos, "cos", _F32),
            (sin, "sin", _F32), (slot_pos, "slot_pos", _I32)))
    B, max_pages, page_size, num_pages, Hkv = _paged(kpages, vpages, block_table, q_start, lens)
    T = k.shape[0]
    if k.shape != (T, Hkv, HEAD_DIM) or v.shape != k.shape:
        raise ValueError("k and v must be [T, Hkv, 128]")
    rows = half = 0
    if cos is not None:
        if cos.dim() != 2 or sin.shape != cos.shape or 2 * cos.shape[1] > HEAD_DIM:
            raise ValueError("cos and sin must be [rows, rot/2] with rot <= 128")
        rows, half = cos.shape
    if positions is not None and positions.shape != (T,):
        raise ValueError("positions must be [T]")
    Hq = q_t = q_h = o_t = o_h = 0
    if q is not None:
        if q.shape[0] != T or q.shape[2] != HEAD_DIM:
            raise ValueError("q must be [T, Hq, 128]")
        if q_out.shape != q.shape:
            raise ValueError("q_out must have q's shape")
        Hq, q_t, q_h, o_t, o_h = q.shape[1], q.stride(0), q.stride(1), q_out.stride(0), q_out.stride(1)
    if slot_pos is not None and slot_pos.shape != (B, Hkv, max_pages * page_size):
        raise ValueError("slot_pos must be [B, Hkv, max_pages * page_size]")
    _call(dev, "gqa_kv_extend_bf16", 0.0, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
          kpages.data_ptr(), vpages.data_ptr(), block_table.data_ptr(), max_pages, page_size, num_pages, q_start.data_ptr(),
          lens.data_ptr(), 0 if positions is None else positions.data_ptr(), 0 if cos is None else cos.data_ptr(),
          0 if sin is None else sin.data_ptr(), rows, 2 * half, 0 if q is None else q.data_ptr(), q_t, q_h,
          0 if q is None else q_out.data_ptr(), o_t, o_h, 0 if slot_pos is None else slot_pos.data_ptr(), B, T, Hq,
          Hkv, HEAD_DIM, GQA_FLAG_INTERLEAVED if interleaved else 0)
    return q_out


def attend_chunk_workspace_bytes(T: int, Hq: int, Hkv: int) -> int:
    return int(_lib.load().gqa_attend_chunk_workspace_size(T, Hq, Hkv))


def attend_chunk(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor,
                 q_start: torch.Tensor, lens: torch.Tensor, *, causal: bool = True, scale: float | None = None,
                 max_q_len: int = 0, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a ragged chunk of new tokens, q [T, Hq, 128] (rotated), over the pages
    that already hold their keys and values: token i of sequence b sees its slots up to
    its own (``causal``) or all lens[b].  ``lse`` (float32 [T, Hq]) receives the natural
    log of the softmax's sum.  ``max_q_len``: the longest sequence's number of new tokens
    where the caller knows it, a hint that only sizes the second launch.  Tokens that see no
    slot give zeros and -inf.  The last bits of the output depend on whether ``lse`` is given
    (some exponentials are coarser without, by 7.5e-5 at most).  V rows are expected to be
    finite: a NaN or infinity can reach earlier tokens of its sequence through a weight of zero."""
    dev = _index(q, "q")
    out = torch.empty(q.shape, dtype=_BF16, device=q.device) if out is None else out
    _check(dev, ((q, "q", _BF16), (out, "out", _BF16)),
           ((kpages, "kpages", _BF16), (vpages, "vpages", _BF16), (block_table, "block_table", _I32),
            (q_start, "q_start", _I32), (lens, "lens", _I32), (lse, "lse", _F32)))
    B, max_pages, page_size, num_pages, Hkv = _paged(kpages, vpages, block_table, q_start, lens)
    T, Hq, d = q.shape
    if d != HEAD_DIM:
        raise ValueError("q must be [T, Hq, 128]")
    if out.shape != q.shape:
        raise ValueError("out must have q's shape")
    if lse is not None and lse.shape != (T, Hq):
        raise ValueError("lse must be [T, Hq]")
    q = _no_broadcast(q)
    workspace = _workspace(workspace, attend_chunk_workspace_bytes(T, Hq, Hkv), dev)
    _call(dev, "gqa_attend_chunk_bf16", _SCALE if scale is None else scale, q.data_ptr(), q.stride(0), q.stride(1), kpages.data_ptr(), vpages.data_ptr(),
          block_table.data_ptr(), max_pages, page_size, num_pages, q_start.data_ptr(), lens.data_ptr(), out.data_ptr(),
          out.stride(0), out.stride(1), 0 if lse is None else lse.data_ptr(), workspace.data_ptr(),
          workspace.numel() * workspace.element_size(), B, T, Hq, Hkv, d, max_q_len, GQA_FLAG_CAUSAL if causal else 0)
    return out


def attn_weight_sums_workspace_bytes() -> int:
    return int(_lib.load().gqa_attn_weight_sums_workspace_size())


def attn_weight_sums(q: torch.Tensor, kpages: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor,
                     lens: torch.Tensor, lse: torch.Tensor, acc: torch.Tensor, *, causal: bool = True,
                     scale: float | None = None, max_q_len: int = 0, acc_out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Add each cached slot's attention weight from this chunk: acc_out[b, h, j] = acc[b, h, j]
    (zero for slots the chunk wrote) + the sum of exp(q . k_j * scale - lse) over the
    group's query heads and the chunk's tokens that see slot j.  acc, acc_out float32
    [B, Hkv, capacity]; entries at lens[b] and above are left alone; acc_out defaults to
    acc (in place).  q, q_start, lens and ``lse`` are those of ``attend_chunk``, whose
    ``max_q_len`` is accepted too (and not needed)."""
    if max_q_len < 0:
        raise ValueError("max_q_len must not be negative")
    dev = _index(q, "q")
    acc_out = acc if acc_out is None else acc_out
    _check(dev, ((q, "q", _BF16),),
           ((kpages, "kpages", _BF16), (block_table, "block_table", _I32), (q_start, "q_start", _I32), (lens, "lens", _I32),
            (lse, "lse", _F32), (acc, "acc", _F32), (acc_out, "acc_out", _F32)))
    B, max_pages, page_size, num_pages, Hkv = _paged(kpages, None, block_table, q_start, lens)
    T, Hq, d = q.shape
    if d != HEAD_DIM:
        raise ValueError("q must be [T, Hq, 128]")
    if lse.shape != (T, Hq):
        raise ValueError("lse must be [T, Hq]")
    if acc.shape != (B, Hkv, max_pages * page_size) or acc_out.shape != acc.shape:
        raise ValueError("acc and acc_out must be [B, Hkv, max_pages * page_size]")
    q = _no_broadcast(q)
    workspace = _workspace(workspace, attn_weight_sums_workspace_bytes(), dev)
    _call(dev, "gqa_attn_weight_sums_f32", _SCALE if scale is None else scale, q.data_ptr(), q.stride(0), q.stride(1), kpages.data_ptr(), block_table.data_ptr(),
          max_pages, page_size, num_pages, q_start.data_ptr(), lens.data_ptr(), lse.data_ptr(), acc.data_ptr(),
          acc_out.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(), B, T, Hq, Hkv, d,
          GQA_FLAG_CAUSAL if causal else 0)
    return acc_out


def kv_evict_workspace_bytes(B: int, Hkv: int, budget: int, capacity: int | None = None) -> int:
    """Bytes that a call with this budget needs: for `capacity` slots a sequence, else for any capacity."""
    rows = budget if capacity is None else min(budget, max(capacity - budget, 0))
    return int(_lib.load().gqa_kv_evict_workspace_size(B, Hkv, rows))


def kv_evict(kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
             acc: torch.Tensor, slot_pos: torch.Tensor, next_pos: torch.Tensor, budget: int, *, recent: int = 0,
             sink: int = 0, acc_out: torch.Tensor | None = None, slot_pos_out: torch.Tensor | None = None,
             lens_out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> None:
    """Keep min(lens[b], budget) slots of every (sequence, kv head): those that hold one of
    the first ``sink`` positions or of the last ``recent`` before next_pos[b] (int32 [B]),
    then those with the largest ``acc``, equal ones by the lower slot.  The i-th slot
    below the new length that goes receives the i-th kept one above it; K and V rows move
    in place, so a sequence that is cut may share no page with another.  acc, slot_pos
    [B, Hkv, capacity] (float32, int32) follow into acc_out, slot_pos_out, the lengths into
    lens_out; each defaults to its input."""
    dev = _index(kpages, "kpages")
    acc_out = acc if acc_out is None else acc_out
    slot_pos_out = slot_pos if slot_pos_out is None else slot_pos_out
    lens_out = lens if lens_out is None else lens_out
    _check(dev, (), ((kpages, "kpages", _BF16), (vpages, "vpages", _BF16), (block_table, "block_table", _I32),
                     (lens, "lens", _I32), (acc, "acc", _F32), (acc_out, "acc_out", _F32), (slot_pos, "slot_pos", _I32),
                     (slot_pos_out, "slot_pos_out", _I32), (next_pos, "next_pos", _I32), (lens_out, "lens_out", _I32)))
    B, max_pages, page_size, num_pages, Hkv = _paged(kpages, vpages, block_table, None, lens)
    shape = (B, Hkv, max_pages * page_size)
    if acc.shape != shape or acc_out.shape != shape or slot_pos.shape != shape or slot_pos_out.shape != shape:
        raise ValueError("acc, acc_out, slot_pos and slot_pos_out must be [B, Hkv, max_pages * page_size]")
    if next_pos.shape != (B,) or lens_out.shape != (B,):
        raise ValueError("next_pos and lens_out must be [B]")
    workspace = _workspace(workspace, kv_evict_workspace_bytes(B, Hkv, budget, shape[2]), dev)
    _call(dev, "gqa_kv_evict_bf16", 0.0, kpages.data_ptr(), vpages.data_ptr(), block_table.data_ptr(), max_pages, page_size,
          num_pages, lens.data_ptr(), lens_out.data_ptr(), acc.data_ptr(), acc_out.data_ptr(), slot_pos.data_ptr(),
          slot_pos_out.data_ptr(), next_pos.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
          B, Hkv, HEAD_DIM, budget, recent, sink)


def linear(x: torch.Tensor, w: torch.Tensor, *, out_f32: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16(x @ w^T) (or the fp32 sums with ``out_f32``) for x [..., K], w [N, K] in the
    HF [out, in] layout (golden projections, llama3_attention_golden_model.py:149-151, :194)."""
    _need(x, "x")
    _need(w, "w")
    K = x.shape[-1]
    if w.dim() != 2 or w.shape[1] != K:
        raise ValueError("w must be [N, K] with K = x.shape[-1]")
    N, M = w.shape[0], x.numel() // K
    odt = torch.float32 if out_f32 else torch.bfloat16
    out = torch.empty(*x.shape[:-1], N, dtype=odt, device=x.device) if out is None else out
    _need(out, "out", odt)
    if out.numel() != M * N:
        raise ValueError("out has the wrong size")
    check(_lib.load().gqa_gemm_bf16(_ptr(x), _ptr(w), _ptr(out), M, N, K, K, K, N,
                                    GQA_GEMM_OUT_F32 if out_f32 else 0, _stream(x.device)), "gqa_gemm_bf16")
    return out


def qkv_proj(h: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor,
             cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *, rope_q: bool = False,
             rope_k: bool = False, pos0: int = 0, head_dim: int = HEAD_DIM,
             out: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None):
    """Fused q/k/v projection (one launch): h [S, hidden] or [B, S, hidden] -> head-major
    q [B?, Hq, S, 128], k/v [B?, Hkv, S, 128] = bf16(h @ W^T) viewed per head
    (golden :149-155); q / k rotated at positions pos0 + s when rope_q / rope_k (:162-164)."""
    for t, n in ((h, "h"), (wq, "wq"), (wk, "wk"), (wv, "wv")):
        _need(t, n)
    batched = h.dim() == 3
    B, S, hidden = (h.shape if batched else (1, *h.shape))
    Hq, Hkv = wq.shape[0] // head_dim, wk.shape[0] // head_dim
    if wq.shape != (Hq * head_dim, hidden) or wk.shape != (Hkv * head_dim, hidden) or wv.shape != wk.shape:
        raise ValueError("weights must be [H*head_dim, hidden]")
    lead = (B,) if batched else ()
    if out is None:
        q = torch.empty(*lead, Hq, S, head_dim, dtype=torch.bfloat16, device=h.device)
        k = torch.empty(*lead, Hkv, S, head_dim, dtype=torch.bfloat16, device=h.device)
        v = torch.empty_like(k)
    else:
        q, k, v = out
    flags = (GQA_FLAG_ROPE_Q if rope_q else 0) | (GQA_FLAG_ROPE_K if rope_k else 0)
    if flags:
        if cos is None or sin is None:
            raise ValueError("rope needs cos/sin tables")
        _need(cos, "cos")
        _need(sin, "sin")
        if cos.shape[0] < pos0 + S:
            raise ValueError("rope table too short")
    cp = _ptr(cos) if flags else None
    sp = _ptr(sin) if flags else None
    check(_lib.load().gqa_qkv_proj_bf16(_ptr(h), _ptr(wq), _ptr(wk), _ptr(wv), _ptr(q), _ptr(k), _ptr(v), cp, sp,
                                        B, S, hidden, Hq, Hkv, head_dim, pos0, flags, _stream(h.device)),
          "gqa_qkv_proj_bf16")
    return q, k, v


def o_proj(attn: torch.Tensor, wo: torch.Tensor, *, head_begin: int = 0, out_f32: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """o_proj straight from the head-major attention output attn [B?, H, S, 128]:
    out [B?, S, N] = concat_h(attn) @ wo[:, head_begin*128 : (head_begin+H)*128]^T (golden :193-194)."""
    _need(attn, "attn")
    _need(wo, "wo")
    a4 = _bhsd(attn, "attn")
    B, H, S, d = a4.shape
    N, width = wo.shape
    if (head_begin + H) * d > width:
        raise ValueError("wo has fewer input columns than the heads need")
    odt = torch.float32 if out_f32 else torch.bfloat16
    shape = (B, S, N) if attn.dim() == 4 else (S, N)
    out = torch.empty(shape, dtype=odt, device=attn.device) if out is None else out
    _need(out, "out", odt)
    w_ptr = _ptr(wo) + head_begin * d * wo.element_size()
    check(_lib.load().gqa_o_proj_bf16(_ptr(attn), w_ptr, _ptr(out), B, S, H, d, N, width,
                                      GQA_GEMM_OUT_F32 if out_f32 else 0, _stream(attn.device)), "gqa_o_proj_bf16")
    return out


def o_proj_rows(attn: torch.Tensor, wo: torch.Tensor, out: torch.Tensor, s0: int, s_count: int, *,
                head_begin: int = 0, out_f32: bool = False, max_ctas: int = 0) -> torch.Tensor:
    """Rows [s0, s0+s_count) of ``o_proj`` for one sequence: attn [H, S, 128] (or
    [1, H, S, 128]) into the full-size ``out`` [S, N] (or [1, S, N]); the other rows are
    left alone.  ``max_ctas`` > 0 caps the GEMM's persistent grid."""
    _need(attn, "attn")
    _need(wo, "wo")
    a4 = _bhsd(attn, "attn")
    B, H, S, d = a4.shape
    if B != 1:
        raise ValueError("o_proj_rows takes one sequence")
    N, width = wo.shape
    if (head_begin + H) * d > width:
        raise ValueError("wo has fewer input columns than the heads need")
    odt = torch.float32 if out_f32 else torch.bfloat16
    _need(out, "out", odt)
    if out.numel() != S * N:
        raise ValueError("out must hold all S x N rows")
    w_ptr = _ptr(wo) + head_begin * d * wo.element_size()
    check(_lib.load().gqa_o_proj_rows_bf16(_ptr(attn), w_ptr, _ptr(out), S, s0, s_count, H, d, N, width, max_ctas,
                                           GQA_GEMM_OUT_F32 if out_f32 else 0, _stream(attn.device)),
          "gqa_o_proj_rows_bf16")
    return out


def cast_bf16(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Round an fp32 tensor to bf16 (RNE), e.g. all-reduced o_proj partials."""
    _need(x, "x", torch.float32)
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device) if out is None else out
    _need(out, "out")
    check(_lib.load().gqa_cast_f32_bf16(_ptr(x), _ptr(out), x.numel(), _stream(x.device)), "gqa_cast_f32_bf16")
    return out


def device_check(device=None) -> None:
    """Synchronize and raise if any kernel's bounded wait expired since the last check."""
    device = torch.device(device or "cuda")
    site = ctypes_int()
    rc = _lib.load().gqa_device_check(_stream(device), site)
    if rc != 0:
        raise GqaError(rc, f"device check (site 0x{site.value:x})")


def ctypes_int():
    import ctypes
    return ctypes.c_int(0)


__all__ = ["rope_cache", "rope", "scores", "mask", "attention_mask_words", "softmax", "pv", "prefill", "decode",
           "decode_workspace_bytes", "device_check", "default_scale", "GqaError", "rope_inv_freq", "rope_table",
           "rope_positions", "kv_extend", "attend_chunk", "attend_chunk_workspace_bytes", "attn_weight_sums",
           "attn_weight_sums_workspace_bytes", "kv_evict",
           "kv_evict_workspace_bytes"]
