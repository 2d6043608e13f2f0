"""Torch-facing wrappers of the libhca_b200 kernels.

Names, argument meaning and return conventions mirror the reference ops the
kernels replace (cited per function).  Tensors must be CUDA tensors; every
call is stream-ordered on ``torch.cuda.current_stream()`` and allocates
only its documented outputs.  A failing status raises ``HcaError``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import call, lib

FP8 = torch.float8_e4m3fn


def _s() -> int:
    return torch.cuda.current_stream().cuda_stream


def _p(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_cuda(*ts: torch.Tensor | None) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("libhca_b200 ops take CUDA tensors")


# ---------------------------------------------------------------------------
# metadata
# ---------------------------------------------------------------------------


def token_to_req_indices(query_start_loc: torch.Tensor, num_tokens: int,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Device ``repeat_interleave(arange(R), query_lens)``
    (``V/v1/attention/backends/mla/sparse_swa.py:286-294``)."""
    _check_cuda(query_start_loc)
    out = out if out is not None else torch.empty(num_tokens, dtype=torch.int32, device=query_start_loc.device)
    call("hca_token_to_req", _p(out), _p(query_start_loc), query_start_loc.numel() - 1, num_tokens, _s())
    return out[:num_tokens]


def slot_mapping(query_start_loc, seq_lens, block_table, block_size: int, num_tokens: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Per-token slot in a paged cache with ``block_size``-token pages."""
    _check_cuda(query_start_loc, seq_lens, block_table)
    out = out if out is not None else torch.empty(num_tokens, dtype=torch.int64, device=block_table.device)
    call("hca_slot_mapping", _p(out), _p(query_start_loc), _p(seq_lens), _p(block_table),
         block_table.stride(0), block_table.shape[0], block_size, _s())
    return out[:num_tokens]


def get_compressed_slot_mapping(num_tokens: int, query_start_loc, seq_lens, block_table,
                                block_size: int, compress_ratio: int,
                                out: torch.Tensor | None = None) -> torch.Tensor:
    """``V/v1/attention/backends/mla/compressor_utils.py:53-86``."""
    _check_cuda(query_start_loc, seq_lens, block_table)
    if out is None:
        out = torch.empty(num_tokens, dtype=torch.int64, device=block_table.device)
    call("hca_compressed_slot_mapping", _p(out), out.numel(), _p(query_start_loc), _p(seq_lens),
         _p(block_table), block_table.stride(0), block_table.shape[0], block_size, compress_ratio, _s())
    return out[:num_tokens]


def compute_swa_indices_and_lens(indices: torch.Tensor, lens: torch.Tensor, num_decode_tokens: int,
                                 window_size: int, query_start_loc, seq_lens, token_to_req,
                                 is_valid_token, block_table, block_size: int) -> None:
    """Fills the builder's persistent ``decode_swa_indices [max, W]`` and
    ``decode_swa_lens [max]`` (``V/v1/attention/backends/mla/sparse_swa.py:296-314,449-503``)."""
    _check_cuda(indices, lens, query_start_loc, seq_lens, token_to_req, is_valid_token, block_table)
    idx2 = indices.view(indices.shape[0], -1)
    call("hca_swa_indices_and_lens", _p(idx2), idx2.stride(0), _p(lens), lens.numel(),
         num_decode_tokens, window_size, _p(query_start_loc), _p(seq_lens), _p(token_to_req),
         _p(is_valid_token.view(torch.uint8)), _p(block_table), block_table.stride(0), block_size, _s())


def build_c128a_topk_metadata(positions, compress_ratio: int, num_decode_tokens: int,
                              token_to_req_indices, block_table, block_size: int, slot_mapping_,
                              global_decode_buffer, decode_lens_buffer, prefill_buffer,
                              max_compressed_tokens: int = 8192):
    """``V/v1/attention/backends/mla/flashmla_sparse.py:1032-1080``; returns
    ``(global_decode, decode_lens, prefill_local)`` slices of the buffers."""
    _check_cuda(positions, token_to_req_indices, block_table, slot_mapping_)
    n = positions.shape[0]
    call("hca_c128a_topk_metadata", _p(global_decode_buffer), global_decode_buffer.stride(0),
         _p(decode_lens_buffer), _p(prefill_buffer), prefill_buffer.stride(0), _p(positions), n,
         compress_ratio, max_compressed_tokens, num_decode_tokens, _p(token_to_req_indices),
         _p(block_table), block_table.stride(0), block_size, _p(slot_mapping_), _s())
    return (global_decode_buffer[:num_decode_tokens], decode_lens_buffer[:num_decode_tokens],
            prefill_buffer[: n - num_decode_tokens])


def compute_prefill_gather_lens(seq_lens, query_start_loc, num_prefills: int, num_decodes: int,
                                window_size: int) -> torch.Tensor:
    """``gather_len = q_len + min(prefix, W - 1)``
    (``V/v1/attention/backends/mla/sparse_swa.py:422-446``)."""
    out = torch.empty(num_prefills, dtype=torch.int32, device=seq_lens.device)
    call("hca_prefill_gather_lens", _p(out), _p(seq_lens), _p(query_start_loc), num_prefills,
         num_decodes, window_size, _s())
    return out


def combine_topk_swa_indices(topk_indices, query_start_loc, seq_lens, gather_lens, window_size: int,
                             compress_ratio: int, topk: int, M: int, N: int):
    """``V/models/deepseek_v4/common/ops/cache_utils.py:476-519``."""
    num_tokens = topk_indices.shape[0]
    width = (topk + window_size + 127) // 128 * 128
    comb = torch.empty((num_tokens, width), dtype=torch.int32, device=topk_indices.device)
    lens = torch.empty(num_tokens, dtype=torch.int32, device=topk_indices.device)
    call("hca_combine_topk_swa_indices", _p(comb), comb.stride(0), width, _p(lens), _p(topk_indices),
         topk_indices.stride(0), _p(query_start_loc), _p(seq_lens), _p(gather_lens),
         seq_lens.shape[0], num_tokens, window_size, compress_ratio, topk, M, N, _s())
    return comb, lens


# ---------------------------------------------------------------------------
# norms, cache write, compressor
# ---------------------------------------------------------------------------


def fused_q_kv_rmsnorm(qr, kv, q_weight, kv_weight, eps: float):
    """``V/models/deepseek_v4/common/ops/fused_qk_rmsnorm.py:57-96``."""
    _check_cuda(qr, kv, q_weight, kv_weight)
    qo, ko = torch.empty_like(qr), torch.empty_like(kv)
    if qr.shape[0]:
        call("hca_qk_rmsnorm", _p(qo), qo.stride(0), _p(qr), qr.stride(0), _p(q_weight), qr.shape[1],
             _p(ko), ko.stride(0), _p(kv), kv.stride(0), _p(kv_weight), kv.shape[1], qr.shape[0],
             eps, _s())
    return qo, ko


def fused_qnorm_rope_kv_insert(q, kv, swa_kv_cache, slot_mapping_, positions, cos_sin_cache,
                               padded_heads: int, eps: float, block_size: int, rope_dim: int = 64,
                               out: torch.Tensor | None = None) -> torch.Tensor:
    """Replacement of ``torch.ops._C.fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert``
    (``V/models/deepseek_v4/attention.py:497-542``); returns the padded q."""
    _check_cuda(q, kv, swa_kv_cache, slot_mapping_, positions, cos_sin_cache)
    t, h, d = q.shape
    if out is None:
        out = torch.empty((t, padded_heads, d), dtype=q.dtype, device=q.device)
    n = slot_mapping_.shape[0]
    if n:
        call("hca_qnorm_rope_kv_insert", _p(out), out.stride(0), out.stride(1), padded_heads, _p(q),
             q.stride(0), q.stride(1), h, _p(kv), kv.stride(0), _p(swa_kv_cache), block_size,
             swa_kv_cache.stride(0), _p(slot_mapping_), _p(positions), _p(cos_sin_cache),
             cos_sin_cache.stride(0), n, d, rope_dim, eps, _s())
    return out


def quantize_and_insert_k_cache(k, k_cache, slot_mapping_, block_size: int = 64, rope_dim: int = 64):
    """``V/models/deepseek_v4/common/ops/cache_utils.py:142-194``."""
    _check_cuda(k, k_cache, slot_mapping_)
    n = slot_mapping_.shape[0]
    if n:
        call("hca_quantize_insert_k", _p(k_cache), block_size, k_cache.stride(0), _p(k), k.stride(0),
             _p(slot_mapping_), n, k.shape[1], rope_dim, _s())


def dequantize_and_gather_k_cache(out, k_cache, seq_lens, gather_lens, block_table, block_size: int,
                                  offset: int, rope_dim: int = 64) -> None:
    """``V/models/deepseek_v4/common/ops/cache_utils.py:355-380``."""
    _check_cuda(out, k_cache, seq_lens, block_table)
    call("hca_dequantize_gather_k", _p(out), out.stride(0), out.stride(1), _p(k_cache), block_size,
         k_cache.stride(0), _p(seq_lens), _p(gather_lens), _p(block_table), block_table.stride(0),
         seq_lens.shape[0], offset, out.shape[-1], rope_dim, _s())


def save_partial_states(kv, score, ape, positions, state_cache, slot_mapping_, block_size: int,
                        state_width: int, compress_ratio: int) -> None:
    """``V/models/deepseek_v4/common/ops/save_partial_states.py:9-45``."""
    _check_cuda(kv, score, ape, positions, state_cache, slot_mapping_)
    n = slot_mapping_.shape[0]
    if n:
        call("hca_save_partial_states", _p(state_cache), state_cache.stride(0), state_cache.stride(1),
             _p(kv), kv.stride(0), _p(score), score.stride(0), _p(ape), ape.stride(0), _p(positions),
             _p(slot_mapping_), n, block_size, kv.shape[-1], state_width, compress_ratio, _s())


def compress_norm_rope_store(state_cache, num_actual: int, token_to_req_indices, positions,
                             slot_mapping_, block_table, block_size: int, state_width: int,
                             cos_sin_cache, kv_cache, kv_slot_mapping, kv_block_size: int,
                             head_dim: int, rope_head_dim: int, compress_ratio: int,
                             rms_norm_weight, rms_norm_eps: float) -> None:
    """``compress_norm_rope_store_{triton,cutedsl}``
    (``V/models/deepseek_v4/common/ops/fused_compress_quant_cache.py:34-109``)."""
    _check_cuda(state_cache, token_to_req_indices, positions, slot_mapping_, block_table,
                cos_sin_cache, kv_cache, kv_slot_mapping, rms_norm_weight)
    if num_actual:
        call("hca_compress_norm_rope_store", _p(state_cache), state_cache.stride(0),
             state_cache.stride(1), state_width, _p(token_to_req_indices), _p(positions),
             _p(slot_mapping_), _p(block_table), block_table.stride(0), block_size,
             _p(rms_norm_weight), rms_norm_eps, _p(cos_sin_cache), cos_sin_cache.stride(0),
             _p(kv_cache), _p(kv_slot_mapping), kv_block_size, kv_cache.stride(0), num_actual,
             head_dim, rope_head_dim, compress_ratio, _s())


def decode_prep(q, kv, kv_score, ape, positions, cos_sin_cache, swa_kv_cache, swa_slot_mapping,
                swa_block_size: int, state_cache, state_slot_mapping, state_block_table, state_block_size: int,
                kv_cache, kv_slot_mapping, kv_block_size: int, rms_norm_weight, query_start_loc,
                token_to_req_indices, num_reqs: int, padded_heads: int, eps: float, compress_ratio: int,
                rope_dim: int = 64, out: torch.Tensor | None = None) -> torch.Tensor:
    """``fused_qnorm_rope_kv_insert`` + ``save_partial_states`` +
    ``compress_norm_rope_store`` of a decode-shaped batch (request r owns
    tokens ``query_start_loc[r] .. query_start_loc[r + 1]``) in one launch,
    with the same output bytes; returns the padded q.  ``kv_score`` is the
    compressor's fp32 ``[T, 2 D]`` (kv then score)."""
    _check_cuda(q, kv, kv_score, ape, positions, cos_sin_cache, swa_kv_cache, swa_slot_mapping, state_cache,
                state_slot_mapping, state_block_table, kv_cache, kv_slot_mapping, rms_norm_weight,
                query_start_loc, token_to_req_indices)
    t, h, d = q.shape
    if out is None:
        out = torch.empty((t, padded_heads, d), dtype=q.dtype, device=q.device)
    n = swa_slot_mapping.shape[0]
    if n:
        ks, sc = kv_score[:, :d], kv_score[:, d:]
        call("hca_decode_prep", _p(out), out.stride(0), out.stride(1), padded_heads, _p(q), q.stride(0),
             q.stride(1), h, _p(kv), kv.stride(0), _p(swa_kv_cache), swa_block_size, swa_kv_cache.stride(0),
             _p(swa_slot_mapping), _p(positions), _p(cos_sin_cache), cos_sin_cache.stride(0), _p(ks), ks.stride(0),
             _p(sc), sc.stride(0), _p(ape), ape.stride(0), _p(state_cache), state_cache.stride(0),
             state_cache.stride(1), d, state_block_size, _p(state_slot_mapping), _p(state_block_table),
             state_block_table.stride(0), _p(rms_norm_weight), _p(kv_cache), _p(kv_slot_mapping), kv_block_size,
             kv_cache.stride(0), _p(query_start_loc), _p(token_to_req_indices), num_reqs, n, d, rope_dim,
             compress_ratio, eps, _s())
    return out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def set_attention_wait_limit_ns(limit_ns: int) -> None:
    """Limit of every mbarrier wait of the head_dim-128 attention kernel for
    launches made from now on (``< 0``: the default 2 s; ``0``: a wait not
    already satisfied fails at once).  A diagnostic for testing the bounded
    waits; it has no counterpart in the reference."""
    call("hca_set_attention_wait_limit_ns", int(limit_ns))


def device_error(clear: bool = True) -> int:
    """The library's device error word (non-zero if a kernel gave up on a
    bounded wait); synchronous."""
    import ctypes

    v = ctypes.c_int32(0)
    call("hca_device_error", ctypes.addressof(v), 1 if clear else 0)
    return int(v.value)


class DecodeWorkspace:
    """Persistent zero-initialised split-K workspace, one buffer per device.

    A buffer's address is stable once a CUDA graph may hold it: it only
    grows while no stream on its device is capturing (a grown buffer would
    free the one a captured graph still points at); a request for more than
    it holds during capture raises instead.  Size it before capture by one
    eager call with the largest shapes (or ``reserve``)."""

    def __init__(self):
        self.bufs: dict[int, torch.Tensor] = {}

    def reserve(self, nbytes: int, device) -> None:
        self.get(nbytes, device)

    def get(self, nbytes: int, device) -> torch.Tensor | None:
        if nbytes == 0:
            return None
        device = torch.device(device)
        idx = device.index if device.index is not None else torch.cuda.current_device()
        buf = self.bufs.get(idx)
        if buf is None or buf.numel() < nbytes:
            if torch.cuda.is_current_stream_capturing():
                have = 0 if buf is None else buf.numel()
                raise RuntimeError(f"decode workspace on cuda:{idx} holds {have} bytes, {nbytes} needed while a "
                                   "CUDA graph is being captured; size it with an eager call (or reserve) first")
            buf = torch.zeros(nbytes, dtype=torch.uint8, device=torch.device("cuda", idx))
            self.bufs[idx] = buf
        return buf


_WS = DecodeWorkspace()


def decode_schedule(group_starts, num_tokens: int, swa_lens, comp_lens, max_items: int, out=None):
    """Per-step decode work list (the role of FlashMLA's ``get_mla_metadata``
    tile-scheduler metadata): ``int32[hca_decode_schedule_ints]``, valid for
    every layer of the step.  ``max_items`` = one wave of CTAs (the SM count,
    at least the number of groups)."""
    _check_cuda(swa_lens)
    num_groups = num_tokens if group_starts is None else group_starts.numel() - 1
    n = lib().hca_decode_schedule_ints(num_groups, max_items)
    if n <= 0:
        raise ValueError(f"decode schedule: max_items={max_items} must cover num_groups={num_groups}")
    if out is None or out.numel() != n:
        out = torch.empty(n, dtype=torch.int32, device=swa_lens.device)
    call("hca_decode_schedule", _p(out), max_items, _p(group_starts), num_groups, num_tokens, _p(swa_lens),
         _p(comp_lens), _s())
    return out


def sparse_decode(q, swa_cache, swa_block_size: int, swa_indices, swa_lens, comp_cache,
                  comp_block_size: int, comp_indices, comp_lens, softmax_scale: float, attn_sink,
                  out=None, group_starts=None, max_group_tokens: int = 1, num_splits: int = 1,
                  lse=None, rope_dim: int = 64, workspace: DecodeWorkspace | None = None,
                  schedule=None, max_items: int = 0):
    """Replacement of ``flash_mla_with_kvcache`` for the HCA decode call
    (``V/models/deepseek_v4/nvidia/flashmla.py:286-302``).  ``q`` is
    ``[T, H, D]`` bf16; ``swa_indices``/``comp_indices`` are the builders'
    ``[T, W]`` / ``[T, C]`` int32 tables (any extra middle dim of size 1 is
    accepted); ``group_starts`` groups consecutive-position tokens of one
    request.  With ``schedule`` (from ``decode_schedule``, same
    ``max_items``) the CTAs follow its balanced work list and ``num_splits``
    is unused; otherwise every group gets ``num_splits`` even splits."""
    _check_cuda(q, swa_cache, swa_indices, swa_lens)
    t, h, d = q.shape
    if out is None:
        out = torch.empty_like(q)
    si = swa_indices.reshape(swa_indices.shape[0], -1)
    ci = comp_indices.reshape(comp_indices.shape[0], -1) if comp_indices is not None else None
    num_groups = t if group_starts is None else group_starts.numel() - 1
    ws = None
    nbytes = 0
    slots = (1, max_items) if schedule is not None else (num_groups, num_splits)
    if slots[1] > 1:
        nbytes = lib().hca_sparse_decode_workspace_bytes(slots[0], max_group_tokens, h, d, slots[1])
        ws = (workspace or _WS).get(nbytes, q.device)
    common = (_p(out), out.stride(0), out.stride(1), _p(lse), _p(q), q.stride(0),
              q.stride(1), t, h, d, rope_dim, _p(swa_cache), swa_block_size, swa_cache.stride(0), _p(si),
              si.stride(0), _p(swa_lens), _p(comp_cache), comp_block_size,
              comp_cache.stride(0) if comp_cache is not None else 0, _p(ci),
              ci.stride(0) if ci is not None else 0, _p(comp_lens), _p(group_starts), num_groups,
              max_group_tokens, softmax_scale, _p(attn_sink))
    if schedule is not None:
        call("hca_sparse_decode_scheduled", *common, _p(schedule), max_items, _p(ws), nbytes, _s())
    else:
        call("hca_sparse_decode", *common, num_splits, _p(ws), nbytes, _s())
    return out


def sparse_prefill(q, query_start_loc, seq_lens, swa_cache, swa_block_size: int, swa_block_table,
                   comp_cache, comp_block_size: int, comp_block_table, window: int,
                   compress_ratio: int, softmax_scale: float, attn_sink, out=None,
                   rope_dim: int = 64):
    """Prefill attention straight from the fp8 caches (replaces the gather +
    ``flash_mla_sparse_fwd`` of ``V/models/deepseek_v4/nvidia/flashmla.py:304-424``)."""
    _check_cuda(q, query_start_loc, seq_lens, swa_cache, swa_block_table)
    t, h, d = q.shape
    if out is None:
        out = torch.empty_like(q)
    call("hca_sparse_prefill", _p(out), out.stride(0), out.stride(1), _p(q), q.stride(0), q.stride(1),
         h, d, rope_dim, _p(query_start_loc), _p(seq_lens), seq_lens.shape[0], t, _p(swa_cache),
         swa_block_size, swa_cache.stride(0), _p(swa_block_table), swa_block_table.stride(0),
         _p(comp_cache), comp_block_size, comp_cache.stride(0) if comp_cache is not None else 0,
         _p(comp_block_table), comp_block_table.stride(0) if comp_block_table is not None else 0,
         window, compress_ratio, softmax_scale, _p(attn_sink), _s())
    return out


# ---------------------------------------------------------------------------
# output path
# ---------------------------------------------------------------------------


def _aligned(n: int) -> int:
    return (n + 3) // 4 * 4


def _quant_out(out, scale, n_groups: int, t: int, hpg: int, d: int, device):
    """The ``(data [G, T, HPG*D] e4m3, scale [G, HPG, round_up(T, 4)] int32)``
    buffers of the VHA quant: the caller's or new ones."""
    if out is None:
        out = torch.empty((n_groups, t, hpg * d), dtype=FP8, device=device)
    if scale is None:
        scale = torch.empty((n_groups, hpg, _aligned(t)), dtype=torch.int32, device=device)
    assert out.shape == (n_groups, t, hpg * d) and out.dtype == FP8 and out.is_contiguous()
    assert scale.shape == (n_groups, hpg, _aligned(t)) and scale.dtype == torch.int32 and scale.is_contiguous()
    return out, scale


def vha_inv_rope_fp8_quant(o, mix, positions, cos_sin_cache, n_groups: int, nope_dim: int,
                           rope_dim: int, out=None, scale_out=None):
    """``E/nvidia/attention.py:232-285``: returns ``(data [T, G, HPG*D] e4m3,
    scale [T, G, HPG] int32)`` views with the plugin's strides (of ``out``
    ``[G, T, HPG*D]`` and ``scale_out`` ``[G, HPG, round_up(T, 4)]`` when
    given)."""
    _check_cuda(o, mix, positions, cos_sin_cache)
    t, h, d = o.shape
    assert d == nope_dim + rope_dim and o.stride(-1) == 1
    hpg = h // n_groups
    out, scale = _quant_out(out, scale_out, n_groups, t, hpg, d, o.device)
    if t:
        call("hca_vha_inv_rope_fp8_quant", _p(out), _p(scale), _p(o), o.stride(0), o.stride(1),
             _p(mix), _p(positions), _p(cos_sin_cache), cos_sin_cache.stride(0), t, h, n_groups, d,
             rope_dim, _s())
    return out.transpose(0, 1), scale.permute(2, 0, 1)[:t]


def sparse_decode_vha_fp8_quant(q, swa_cache, swa_block_size: int, swa_indices, swa_lens, comp_cache,
                                comp_block_size: int, comp_indices, comp_lens, softmax_scale: float,
                                attn_sink, group_starts, max_group_tokens: int, schedule, max_items: int,
                                mix, positions, cos_sin_cache, n_groups: int, rope_dim: int = 64,
                                workspace: DecodeWorkspace | None = None, out=None, scale_out=None):
    """Decode attention (scheduled) fused with the VHA mix, inverse RoPE and
    FP8 quant: ``sparse_decode`` followed by ``vha_inv_rope_fp8_quant`` in two
    launches, without the bf16 O round trip.  Returns the same
    ``(data [T, G, HPG*D] e4m3, scale [T, G, HPG] int32)`` views."""
    _check_cuda(q, swa_cache, swa_indices, swa_lens, mix, positions, cos_sin_cache, schedule)
    t, h, d = q.shape
    hpg = h // n_groups
    out, scale = _quant_out(out, scale_out, n_groups, t, hpg, d, q.device)
    if t == 0:
        return out.transpose(0, 1), scale.permute(2, 0, 1)[:t]
    si = swa_indices.reshape(swa_indices.shape[0], -1)
    ci = comp_indices.reshape(comp_indices.shape[0], -1) if comp_indices is not None else None
    num_groups = t if group_starts is None else group_starts.numel() - 1
    nbytes = lib().hca_sparse_decode_vha_workspace_bytes(max_items, max_group_tokens, h, d)
    ws = (workspace or _WS).get(nbytes, q.device)
    call("hca_sparse_decode_vha_fp8_quant", _p(out), _p(scale), _p(q), q.stride(0), q.stride(1), t, h, d,
         rope_dim, _p(swa_cache), swa_block_size, swa_cache.stride(0), _p(si), si.stride(0), _p(swa_lens),
         _p(comp_cache), comp_block_size, comp_cache.stride(0) if comp_cache is not None else 0, _p(ci),
         ci.stride(0) if ci is not None else 0, _p(comp_lens), _p(group_starts), num_groups, max_group_tokens,
         softmax_scale, _p(attn_sink), _p(schedule), max_items, _p(mix), _p(positions), _p(cos_sin_cache),
         cos_sin_cache.stride(0), n_groups, _p(ws), nbytes, _s())
    return out.transpose(0, 1), scale.permute(2, 0, 1)[:t]


def fused_inv_rope_fp8_quant(o, positions, cos_sin_cache, n_groups: int, heads_per_group: int,
                             nope_dim: int = 448, rope_dim: int = 64):
    """``V/models/deepseek_v4/common/ops/fused_inv_rope_fp8_quant.py:138-193``
    with ``tma_aligned_scales=True``: ``(fp8 [T, G, D'], scale [T, G, packs])``."""
    _check_cuda(o, positions, cos_sin_cache)
    t, h, d = o.shape
    dd = heads_per_group * d
    packs = (dd // 128 + 3) // 4
    out = torch.empty((n_groups, t, dd), dtype=FP8, device=o.device)
    al = _aligned(t)
    buf = torch.empty(n_groups * packs * al, dtype=torch.int32, device=o.device)
    if t:
        call("hca_inv_rope_fp8_quant", _p(out), _p(buf), _p(o), o.stride(0), o.stride(1),
             _p(positions), _p(cos_sin_cache), cos_sin_cache.stride(0), t, h, n_groups, d, rope_dim, _s())
    scale = buf.as_strided((n_groups, t, packs), (packs * al, 1, al))
    return out.transpose(0, 1), scale.transpose(0, 1)


def vha_inv_rope(o, mix, positions, cos_sin_cache, rope_dim: int = 64, out=None):
    """``inverse_rope(m @ o)`` in bf16 for the bf16 ``wo_a`` path."""
    _check_cuda(o, positions, cos_sin_cache)
    t, h, d = o.shape
    out = out if out is not None else torch.empty((t, h, d), dtype=o.dtype, device=o.device)
    if t:
        call("hca_vha_inv_rope", _p(out), out.stride(0), out.stride(1), _p(o), o.stride(0),
             o.stride(1), _p(mix), _p(positions), _p(cos_sin_cache), cos_sin_cache.stride(0), t, h, d,
             rope_dim, _s())
    return out


def sigmoid_mul_quant_fp8(x, gate):
    """``E/nvidia/attention.py:330-361``: ``(fp8 [rows, hidden], scale [rows, packs])``."""
    _check_cuda(x, gate)
    rows, hidden = x.shape
    assert gate.shape == x.shape and hidden % 512 == 0
    out = torch.empty((rows, hidden), dtype=FP8, device=x.device)
    packs = hidden // 512
    scale = torch.empty_strided((rows, packs), (1, _aligned(rows)), dtype=torch.int32, device=x.device)
    if rows:
        call("hca_sigmoid_mul_quant_fp8", _p(out), _p(scale), _p(x), x.stride(0), _p(gate),
             gate.stride(0), rows, hidden, _s())
    return out, scale




# split-K partial tiles of the FP8 GEMM (one buffer per device; calls are
# ordered on the current stream)
_GEMM_WS = DecodeWorkspace()


def fp8_grouped_gemm(x, x_scale, w, w_scale, out=None, workspace: DecodeWorkspace | None = None):
    """Block-scaled FP8 GEMM of the output path: the grouped ``wo_a`` einsum
    ``"bhr,hdr->bhd"`` (``V/models/deepseek_v4/attention.py:317-347``) for a
    3-D ``x [T, G, K]`` and ``w [G, N, K]``, or the gated ``wo_b`` linear
    (``E/nvidia/attention.py:364-395``) for a 2-D ``x [T, K]`` and ``w [N, K]``.
    ``x`` e4m3 with the int32 UE8M0 scales the quant kernels write
    (``[T, G, packs]`` or ``[T, packs]``, one or four 128-blocks per int32);
    ``w`` e4m3 with fp32 128 x 128 block scales ``[G, ceil(N/128), K/128]`` (or
    ``[ceil(N/128), K/128]``).  Returns bf16 ``[T, G, N]`` (or ``[T, N]``)."""
    _check_cuda(x, x_scale, w, w_scale)
    flat = x.dim() == 2
    if flat:
        x, x_scale, w, w_scale = x.unsqueeze(1), x_scale.unsqueeze(1), w.unsqueeze(0), w_scale.unsqueeze(0)
    t, g, k = x.shape
    n = w.shape[1]
    assert x.dtype == FP8 and w.dtype == FP8 and x.stride(2) == 1
    assert w.shape == (g, n, k) and w.is_contiguous()
    assert w_scale.dtype == torch.float32 and w_scale.is_contiguous() and w_scale.shape == (g, (n + 127) // 128, k // 128)
    assert x_scale.dtype == torch.int32 and x_scale.shape[:2] == (t, g) and k % 128 == 0
    per_int = (k // 128) // x_scale.shape[2]
    assert per_int in (1, 4) and per_int * x_scale.shape[2] == k // 128
    if out is None:
        out = torch.empty((t, g, n), dtype=torch.bfloat16, device=x.device)
    elif flat:
        out = out.unsqueeze(1)
    assert out.shape == (t, g, n) and out.dtype == torch.bfloat16 and out.stride(2) == 1
    if t:
        nbytes = lib().hca_fp8_grouped_gemm_workspace_bytes(t, g, n, k)
        ws = (workspace or _GEMM_WS).get(nbytes, x.device) if nbytes > 0 else None
        call("hca_fp8_grouped_gemm", _p(out), out.stride(0), out.stride(1) if g > 1 else 0, _p(x), x.stride(0),
             x.stride(1) if g > 1 else 0, _p(x_scale), x_scale.stride(0), x_scale.stride(1) if g > 1 else 0,
             x_scale.stride(2), per_int, _p(w), _p(w_scale), t, g, n, k, _p(ws), nbytes, _s())
    return out.squeeze(1) if flat else out


def quantize_weight_block_fp8(w: torch.Tensor, block: int = 128):
    """Load-time 128 x 128 block FP8 quant of a bf16 weight ``[..., N, K]``:
    power-of-two (UE8M0-valued) fp32 block scales, the format the Blackwell
    DeepGEMM path runs block-FP8 checkpoints in (``E/nvidia/quant_config.py``;
    ``dequantize_block_fp8`` there is its inverse).  Returns ``(w_fp8,
    scale [..., ceil(N/128), K/128])``.  A one-off weight transform, not a
    step of the forward pass."""
    *lead, n, k = w.shape
    assert k % block == 0
    nb = (n + block - 1) // block
    wf = torch.zeros((*lead, nb * block, k), dtype=torch.float32, device=w.device)
    wf[..., :n, :] = w.float()
    blocks = wf.view(*lead, nb, block, k // block, block)
    amax = blocks.abs().amax(dim=(-3, -1)).clamp_min(1e-10)
    e = torch.ceil(torch.log2(amax / 448.0))
    scale = torch.exp2(e)
    q = (blocks / scale[..., :, None, :, None]).clamp(-448.0, 448.0).to(FP8)
    return q.view(*lead, nb * block, k)[..., :n, :].contiguous(), scale.contiguous()


# ---------------------------------------------------------------------------
# the rest of a decode step: products on a few rows, logits
# ---------------------------------------------------------------------------

W4_GROUPS = (32, 64, 128)
_BF16, _FP16, _FP32, _U8, _I32 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int32


def _refuse(what: str):
    raise ValueError(what)


# These operators take microseconds on the GPU, so their checks read each
# attribute once and put no message together before it is needed.


def _device_of(x: torch.Tensor, *ts: torch.Tensor | None) -> int:
    """The device of all the tensors, which has to be the current one."""
    dev = x.get_device()
    if dev < 0 or dev != torch._C._cuda_getDevice():
        _refuse("libhca_b200 ops take CUDA tensors of the current device")
    for t in ts:
        if t is not None and t.get_device() != dev:
            _refuse("libhca_b200 ops take CUDA tensors of the current device")
    return dev


def _stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


def _rows_out(x: torch.Tensor, dev: int, t: int, n: int, out: torch.Tensor) -> int:
    """Row stride of a caller's ``out``."""
    if out.get_device() != dev or out.dtype is not x.dtype or out.shape != (t, n):
        _refuse(f"out must be {x.dtype} [{t}, {n}] on x's device")
    stride, inner = out.stride()
    if (n > 1 and inner != 1) or (t > 1 and stride < n):
        _refuse("out must have contiguous rows that do not overlap")
    return stride


def _check_rows(x: torch.Tensor) -> tuple[int, int, int, int]:
    """``(T, K, row stride, address)`` of a matrix whose rows start on 16 bytes."""
    try:
        t, k = x.shape
    except ValueError:
        _refuse("x must be a matrix")
    stride, inner = x.stride()
    at = x.data_ptr()
    if (inner != 1 and k > 1) or (stride % 8 and t > 1) or at % 16:
        _refuse("x must have contiguous rows that start on 16 bytes")
    return t, k, stride if t > 1 else k + -k % 8, at


def _check_w4(q, s, z, lead: tuple, n: int, k: int, dtype) -> int:
    """Group size of the 4-bit weights ``[*lead, n, k]``."""
    shape = s.shape
    groups = shape[-1] if len(shape) else 0
    if groups == 0 or k % groups or k // groups not in W4_GROUPS:
        _refuse(f"scales must be [..., N, K / group] for a group of {W4_GROUPS}")
    if q.dtype is not _U8 or q.shape != (*lead, n, k // 2) or not q.is_contiguous():
        _refuse(f"4-bit codes must be contiguous uint8 {[*lead, n, k // 2]}")
    if s.dtype is not dtype or shape != (*lead, n, groups) or not s.is_contiguous():
        _refuse(f"scales must be contiguous {dtype} {[*lead, n, groups]}")
    if z is not None and (z.dtype is not _U8 or z.shape != shape or not z.is_contiguous()):
        _refuse("zero points must be contiguous uint8 of the scales' shape")
    return k // groups


def w4_linear(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``x W^T`` for 4-bit weights with group scales and a few rows of ``x``.

    ``x`` ``[T, K]`` bf16 or fp16; ``qweight`` uint8 ``[N, K / 2]`` (low nibble
    = even k); ``scales`` ``[N, K / g]`` of x's type, g = 32, 64 or 128;
    ``zeros`` uint8 ``[N, K / g]`` (None: 8), codes starting on 16 bytes, scales and
    zeros on 4.  ``w = (q - zero) * scale``, sums
    in fp32, one rounding to x's type.  A bf16 ``|x|`` of 2^48 and more counts as
    infinite, below 2^-73 terms lose bits; an infinite or NaN ``x`` makes its own
    row infinite or NaN.  ``out`` must not overlap ``x``.  Right
    for any T, made for up to 16 rows (each 16 more read the weights again; a
    prompt's thousands belong on a dense product)."""
    # in line, as the shortest of these calls take the GPU 4 us
    dev = x.get_device()
    if not -1 < dev == qweight.get_device() == scales.get_device() == torch._C._cuda_getDevice():
        _refuse("libhca_b200 ops take CUDA tensors of the current device")
    dtype = x.dtype
    if dtype is not _BF16 and dtype is not _FP16:
        _refuse(f"x must be bf16 or fp16, got {dtype}")
    try:
        (t, k), (n, half), (rows, groups) = x.shape, qweight.shape, scales.shape
    except ValueError:
        _refuse("x must be [T, K], qweight [N, K / 2] and scales [N, K / g]")
    stride, inner = x.stride()
    at = x.data_ptr()
    if inner != 1 or (stride % 8 and t > 1) or at % 16:
        _refuse("x must have contiguous rows that start on 16 bytes")
    if qweight.dtype is not _U8 or n == 0 or 2 * half != k or not qweight.is_contiguous():
        _refuse(f"4-bit codes must be contiguous uint8 {[n, k // 2]}")
    if scales.dtype is not dtype or rows != n or groups == 0 or k % groups or not scales.is_contiguous():
        _refuse(f"scales must be contiguous {dtype} [{n}, K / g]")
    group = k // groups
    if group not in W4_GROUPS:
        _refuse(f"the group size must be one of {W4_GROUPS}, got {group}")
    if zeros is not None and (zeros.get_device() != dev or zeros.dtype is not _U8 or zeros.shape != (n, groups)
                              or not zeros.is_contiguous()):
        _refuse("zero points must be contiguous uint8 of the scales' shape")
    if t < 2:
        stride = k
    if out is None:
        out, out_stride = x.new_empty(t, n), n
    else:
        out_stride = _rows_out(x, dev, t, n, out)
    if t:
        call("hca_w4_linear", out.data_ptr(), out_stride, at, stride, qweight.data_ptr(), scales.data_ptr(),
             None if zeros is None else zeros.data_ptr(), t, n, k, group, dtype is _FP16, _stream(dev))
    return out


def quantize_weight_w4(w: torch.Tensor, group: int = 128, asymmetric: bool = False, dtype=torch.bfloat16):
    """Load-time 4-bit quant of ``w [..., N, K]`` for ``w4_linear`` and
    ``MoEWeights``: ``(qweight uint8 [..., N, K / 2], scales [..., N, K / g] of
    ``dtype``, zeros uint8 or None)``, nearest codes.  A one-off weight
    transform, not a step of the forward pass."""
    *lead, n, k = w.shape
    if group not in W4_GROUPS or k % group:
        _refuse(f"group size must be one of {W4_GROUPS} and divide K")
    g = w.float().unflatten(-1, (k // group, group))
    if asymmetric:
        low, high = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
        scale = ((high - low) / 15).to(dtype)
        step = torch.where(scale > 0, scale.float(), 1.0)
        zero = torch.round(-low / step).clamp(0, 15)
    else:
        scale = (g.abs().amax(-1) / 7).to(dtype)
        step = torch.where(scale > 0, scale.float(), 1.0)
        zero = torch.full_like(step, 8.0)
    codes = (torch.round(g / step.unsqueeze(-1)) + zero.unsqueeze(-1)).clamp(0, 15).to(torch.uint8).flatten(-2)
    q = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return q.contiguous(), scale.contiguous(), zero.to(torch.uint8).contiguous() if asymmetric else None


class MoEWeights(NamedTuple):
    """Gated MLP weights of a stack of experts (or, without the leading
    dimension, of a shared expert), in one of three formats by ``w13``'s type:

    * bf16: ``w13 [E, 2 I, H]`` (gate rows over up rows), ``w2 [E, H, I]``;
    * e4m3 with fp32 scales of 128 x 128 blocks, ``s13 [E, ceil(2 I / 128),
      ceil(H / 128)]``, ``s2 [E, ceil(H / 128), ceil(I / 128)]``;
    * uint8 4-bit codes ``[E, 2 I, H / 2]``, ``[E, H, I / 2]`` with bf16 group
      scales and optional zero points, as ``w4_linear``.

    With e4m3 and 4-bit weights the layer's input and its gated product have the
    range of ``w4_linear``'s bf16 ``x``: below 2^48."""

    w13: torch.Tensor
    w2: torch.Tensor
    s13: torch.Tensor | None = None
    s2: torch.Tensor | None = None
    z13: torch.Tensor | None = None
    z2: torch.Tensor | None = None


_MOE_FORMATS = {torch.bfloat16: 0, FP8: 1, torch.uint8: 2}


def _moe_weights(w: MoEWeights, lead: tuple, hidden: int, dev: int) -> tuple[int, int, int, tuple]:
    """``(format, group, inner, addresses)`` of checked weights."""
    w13, w2, s13, s2, z13, z2 = w
    fmt = _MOE_FORMATS.get(w13.dtype, -1)
    if fmt < 0 or w2.dtype is not w13.dtype:
        _refuse("expert weights must be bf16, e4m3 or uint8 (4-bit codes), both alike")
    if not w13.get_device() == w2.get_device() == dev:
        _refuse("expert weights must be on x's device")
    shape = w13.shape
    if len(shape) != len(lead) + 2 or shape[-2] % 2 or shape[-2] == 0:
        _refuse(f"w13 must be {[*lead, '2 I', 'H']}")
    inner = shape[-2] // 2
    if fmt == 0:
        if s13 is not None or s2 is not None:
            _refuse("bf16 experts have no scales")
    elif s13 is None or s2 is None:
        _refuse("e4m3 and 4-bit experts need scales")
    elif not s13.get_device() == s2.get_device() == dev:
        _refuse("expert weights must be on x's device")
    zeros = None, None
    if z13 is not None or z2 is not None:
        if fmt != 2:
            _refuse("only 4-bit experts have zero points")
        for z in (z13, z2):
            if z is not None and z.get_device() != dev:
                _refuse("expert weights must be on x's device")
        zeros = _p(z13), _p(z2)
    if fmt == 2:
        group = _check_w4(w13, s13, z13, lead, 2 * inner, hidden, _BF16)
        if _check_w4(w2, s2, z2, lead, hidden, inner, _BF16) != group:
            _refuse("w13 and w2 must have one group size")
        return fmt, group, inner, (w13.data_ptr(), s13.data_ptr(), zeros[0], w2.data_ptr(), s2.data_ptr(), zeros[1])
    if shape != (*lead, 2 * inner, hidden) or w2.shape != (*lead, hidden, inner) or not (w13.is_contiguous() and w2.is_contiguous()):
        _refuse(f"expert weights must be contiguous {[*lead, 2 * inner, hidden]} and {[*lead, hidden, inner]}")
    if fmt == 1:
        for s, n, k in ((s13, 2 * inner, hidden), (s2, hidden, inner)):
            if s.dtype is not _FP32 or s.shape != (*lead, -(-n // 128), -(-k // 128)) or not s.is_contiguous():
                _refuse(f"block scales must be contiguous fp32 {[*lead, -(-n // 128), -(-k // 128)]}")
        return fmt, 0, inner, (w13.data_ptr(), s13.data_ptr(), None, w2.data_ptr(), s2.data_ptr(), None)
    return fmt, 0, inner, (w13.data_ptr(), None, None, w2.data_ptr(), None, None)


_NO_SHARED = (None,) * 6


def _moe_args(hidden: int, dev: int, experts: MoEWeights, shared: MoEWeights | None):
    """Checked ``(format, group, weight addresses, E, I, Is)``."""
    if experts[0].dim() != 3:
        _refuse("w13 must be [E, 2 I, H]")
    num = experts[0].shape[0]
    fmt, group, inner, ptrs = _moe_weights(experts, (num,), hidden, dev)
    if shared is None:
        return fmt, group, ptrs + _NO_SHARED, num, inner, 0
    sfmt, sgroup, shared_inner, more = _moe_weights(shared, (), hidden, dev)
    if (sfmt != fmt or sgroup != group or (shared[4] is None) != (experts[4] is None)
            or (shared[5] is None) != (experts[5] is None)):
        _refuse("the shared expert must have the experts' format")
    return fmt, group, ptrs + more, num, inner, shared_inner


def _moe_rows(x, token_mask, *ts) -> tuple[int, int, int, int, int]:
    """Checked ``(device, T, H, row stride, address)`` of the layer's input."""
    dev = _device_of(x, token_mask, *ts)
    if x.dtype is not _BF16:
        _refuse(f"x must be bf16, got {x.dtype}")
    t, hidden, stride, at = _check_rows(x)
    if token_mask is not None and (token_mask.dtype not in (torch.bool, _U8) or token_mask.shape != (t,)
                                   or not token_mask.is_contiguous()):
        _refuse(f"token_mask must be contiguous bool [{t}]")
    return dev, t, hidden, stride, at


def _router_args(hidden: int, router_weight, router_bias, top_k: int, score: str) -> tuple[int, int, int, int | None, int]:
    """Checked ``(E, address, is fp32, bias address, is sigmoid)``."""
    if score != "softmax" and score != "sigmoid":
        _refuse(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    dtype = router_weight.dtype
    if (router_weight.dim() != 2 or router_weight.shape[1] != hidden or not router_weight.is_contiguous()
            or (dtype is not _BF16 and dtype is not _FP32)):
        _refuse(f"router_weight must be contiguous bf16 or fp32 [E, {hidden}]")
    num = router_weight.shape[0]
    if router_bias is not None and (router_bias.dtype is not _FP32 or router_bias.shape != (num,) or not router_bias.is_contiguous()):
        _refuse(f"router_bias must be contiguous fp32 [{num}]")
    if not 1 <= top_k <= num:
        _refuse(f"top_k must be 1 to {num}, got {top_k}")
    return num, router_weight.data_ptr(), dtype is _FP32, _p(router_bias), score == "sigmoid"


def moe_route(x: torch.Tensor, router_weight: torch.Tensor, top_k: int, *, score: str = "softmax",
              router_bias: torch.Tensor | None = None, renormalize: bool = True, routed_scale: float = 1.0,
              token_mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Router of a mixture-of-experts layer for a few tokens: ``(ids int32
    [T, top_k], weights fp32 [T, top_k])``, largest score first.

    ``x`` bf16 ``[T, H]``; ``router_weight`` ``[E, H]`` bf16 or fp32, products
    in fp32.  Scores are ``softmax`` or ``sigmoid`` of the logits; experts are
    chosen by score + ``router_bias`` (ties to the lower expert) and weighted by
    the score alone, renormalised over the chosen ones if asked for, times
    ``routed_scale``.  Rows that ``token_mask`` (bool ``[T]``) leaves out get
    ids -1 and weights 0.  E <= 512, top_k <= 16, H a multiple of 32."""
    dev, t, hidden, stride, at = _moe_rows(x, token_mask, router_weight, router_bias)
    num, wr, fp32, bias, sigmoid = _router_args(hidden, router_weight, router_bias, top_k, score)
    ids = torch.empty((t, top_k), dtype=_I32, device=x.device)
    weights = torch.empty((t, top_k), dtype=_FP32, device=x.device)
    nbytes = lib().hca_moe_route_workspace_bytes(t, num)
    ws = torch.empty(nbytes, dtype=_U8, device=x.device)
    call("hca_moe_route", ids.data_ptr(), weights.data_ptr(), at, stride, wr, fp32, bias, _p(token_mask), t, num, hidden,
         top_k, sigmoid, renormalize, routed_scale, ws.data_ptr(), nbytes, _stream(dev))
    return ids, weights


def moe_experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, experts: MoEWeights, *,
                shared: MoEWeights | None = None, token_mask: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """Experts of a mixture-of-experts layer for a few tokens: ``y[t] = sum_j
    weights[t, j] W2_e (silu(W1_e x_t) * (W3_e x_t))`` with ``e = ids[t, j]``,
    plus the ``shared`` expert (weight 1).

    ``ids`` int32 ``[T, top_k]`` (ids outside ``[0, E)`` are skipped, as for the
    experts of another rank; an id may repeat), ``weights`` fp32 ``[T, top_k]``.
    Each chosen expert's weights are read once for all its tokens (of 64 at a
    time; again for each 8 or 16 tokens of one expert).  Rows that ``token_mask``
    leaves out come out as 0 and choose nothing.  The gated product, its
    weight included, is kept in two bf16 parts (16 bits); sums are fp32."""
    dev, t, hidden, stride, at = _moe_rows(x, token_mask, ids, weights)
    fmt, group, ptrs, num, inner, shared_inner = _moe_args(hidden, dev, experts, shared)
    if (ids.dtype is not _I32 or ids.dim() != 2 or ids.shape[0] != t or not ids.is_contiguous()
            or weights.dtype is not _FP32 or weights.shape != ids.shape or not weights.is_contiguous()):
        _refuse(f"ids must be contiguous int32 [{t}, top_k] and weights fp32 alike")
    top_k = ids.shape[1]
    if out is None:
        out, out_stride = x.new_empty(t, hidden), hidden
    else:
        out_stride = _rows_out(x, dev, t, hidden, out)
    nbytes = lib().hca_moe_workspace_bytes(t, num, top_k, hidden, inner, shared_inner)
    ws = torch.empty(nbytes, dtype=_U8, device=x.device)
    call("hca_moe_experts", out.data_ptr(), out_stride, at, stride, ids.data_ptr(), weights.data_ptr(), _p(token_mask), fmt,
         group, *ptrs, t, num, hidden, inner, shared_inner, top_k, ws.data_ptr(), nbytes, _stream(dev))
    return out


def moe_decode(x: torch.Tensor, router_weight: torch.Tensor, experts: MoEWeights, top_k: int, *, score: str = "softmax",
               router_bias: torch.Tensor | None = None, renormalize: bool = True, routed_scale: float = 1.0,
               shared: MoEWeights | None = None, token_mask: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """A whole mixture-of-experts layer for a few tokens (``moe_route`` then
    ``moe_experts``) in one call of two launches; ``x`` and the result bf16
    ``[T, H]``.  Its scratch comes from the caching allocator on the current
    stream, so calls on several streams do not meet."""
    dev, t, hidden, stride, at = _moe_rows(x, token_mask, router_weight, router_bias)
    fmt, group, ptrs, num, inner, shared_inner = _moe_args(hidden, dev, experts, shared)
    rows, wr, fp32, bias, sigmoid = _router_args(hidden, router_weight, router_bias, top_k, score)
    if rows != num:
        _refuse(f"router_weight must have the {num} experts' rows")
    if out is None:
        out, out_stride = x.new_empty(t, hidden), hidden
    else:
        out_stride = _rows_out(x, dev, t, hidden, out)
    nbytes = lib().hca_moe_workspace_bytes(t, num, top_k, hidden, inner, shared_inner)
    ws = x.new_empty((nbytes + 1) // 2)
    call("hca_moe_decode", out.data_ptr(), out_stride, at, stride, wr, fp32, bias, sigmoid, renormalize, routed_scale,
         _p(token_mask), fmt, group, *ptrs, t, num, hidden, inner, shared_inner, top_k, ws.data_ptr(), nbytes, _stream(dev))
    return out


_LOGIT_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def apply_logit_penalties(logits: torch.Tensor, token_ids: torch.Tensor | None = None,
                          prompt_lens: torch.Tensor | None = None, seq_lens: torch.Tensor | None = None, *,
                          repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                          presence: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                          bias_values: torch.Tensor | None = None, allowed_bitmask: torch.Tensor | None = None,
                          req_index: torch.Tensor | None = None) -> torch.Tensor:
    """Biases, penalties for repeated tokens and a grammar mask on ``logits
    [rows, V]`` (fp32, bf16 or fp16, contiguous rows), in place; returns them.

    In this order: a biased token's ``x += bias``; a token of the prompt or the
    answer ``x > 0 ? x / repetition : x * repetition``; one that the answer
    holds n times ``x -= frequency * n + presence``; one that the mask does not
    allow ``-inf``.  ``token_ids`` int32 ``[R, >= seq_len]``: row i's prompt is
    ``[0, prompt_lens[i])`` and its answer ``[prompt_lens[i], seq_lens[i])`` of
    request ``req_index[i]`` (int32; None: request i; outside ``[0, R)``: the
    row is left alone), so a request's draft rows can share its tokens.
    ``repetition``/``frequency``/``presence`` fp32 ``[R]``; ``bias_ids`` int32
    and ``bias_values`` fp32 ``[R, M]`` (of an id listed twice the later
    counts); ids outside ``[0, V)``, like -1, are skipped.  ``allowed_bitmask``
    int32 ``[rows, ceil(V / 32)]``, bit ``v % 32`` of word ``v // 32``."""
    dev = logits.get_device()
    if not -1 < dev == torch._C._cuda_getDevice():
        _refuse("libhca_b200 ops take CUDA tensors of the current device")
    kind = _LOGIT_TYPES.get(logits.dtype, -1)
    if kind < 0:
        _refuse(f"logits must be fp32, bf16 or fp16, got {logits.dtype}")
    try:
        rows, vocab = logits.shape
    except ValueError:
        _refuse("logits must be [rows, V]")
    logits_stride, inner = logits.stride()
    if vocab == 0 or (vocab > 1 and inner != 1) or (rows > 1 and logits_stride < vocab):
        _refuse("logits must be [rows, V] with contiguous rows that do not overlap")
    reqs = rows
    for t in (token_ids, repetition, frequency, presence, bias_ids):
        if t is not None:
            if not t.dim():
                _refuse("token_ids, penalties and bias_ids have a row or a value a request")
            reqs = t.shape[0]
            break
    at = [0, 0, 0]  # addresses of the penalties
    for i, t in enumerate((repetition, frequency, presence)):
        if t is not None:
            if t.dtype is not _FP32 or t.shape != (reqs,) or not t.is_contiguous() or t.get_device() != dev:
                _refuse(f"penalties must be contiguous fp32 [{reqs}] on the logits' device")
            at[i] = t.data_ptr()
    index = 0
    if req_index is None:
        if reqs != rows:
            _refuse(f"{reqs} requests for {rows} rows need req_index")
    else:
        if (req_index.dtype is not _I32 or req_index.shape != (rows,) or not req_index.is_contiguous()
                or req_index.get_device() != dev):
            _refuse(f"req_index must be contiguous int32 [{rows}] on the logits' device")
        index = req_index.data_ptr()
    width = stride = tokens = prompts = lens = 0
    if token_ids is not None:
        if token_ids.dtype is not _I32 or token_ids.dim() != 2 or token_ids.shape[0] != reqs or token_ids.get_device() != dev:
            _refuse(f"token_ids must be int32 [{reqs}, L] on the logits' device")
        width = token_ids.shape[1]
        stride, inner = token_ids.stride()
        if width > 1 and inner != 1:
            _refuse("token_ids must have contiguous rows")
        for t in (prompt_lens, seq_lens):
            if t is None or t.dtype is not _I32 or t.shape != (rows,) or not t.is_contiguous() or t.get_device() != dev:
                _refuse(f"prompt_lens and seq_lens must be contiguous int32 [{rows}] on the logits' device")
        tokens, prompts, lens = token_ids.data_ptr(), prompt_lens.data_ptr(), seq_lens.data_ptr()
    bias_width = biases = values = 0
    if bias_ids is not None or bias_values is not None:
        if bias_ids is None or bias_values is None:
            _refuse("bias_ids and bias_values come together")
        if (bias_ids.dtype is not _I32 or bias_ids.dim() != 2 or bias_ids.shape[0] != reqs or not bias_ids.is_contiguous()
                or bias_values.dtype is not _FP32 or bias_values.shape != bias_ids.shape or not bias_values.is_contiguous()
                or not bias_ids.get_device() == bias_values.get_device() == dev):
            _refuse(f"bias_ids must be contiguous int32 [{reqs}, M] and bias_values fp32 alike, on the logits' device")
        bias_width, biases, values = bias_ids.shape[1], bias_ids.data_ptr(), bias_values.data_ptr()
    allowed_stride = allowed = 0
    if allowed_bitmask is not None:
        words = (vocab + 31) // 32
        if (allowed_bitmask.dtype is not _I32 or allowed_bitmask.shape != (rows, words)
                or allowed_bitmask.get_device() != dev):
            _refuse(f"allowed_bitmask must be int32 [{rows}, {words}] on the logits' device")
        allowed_stride, inner = allowed_bitmask.stride()
        if words > 1 and inner != 1:
            _refuse("allowed_bitmask must have contiguous rows")
        allowed = allowed_bitmask.data_ptr()
    call("hca_logit_penalties", logits.data_ptr(), logits_stride, kind, index, reqs, tokens, stride, width, prompts, lens,
         at[0], at[1], at[2], biases, values, bias_width, bias_width, allowed, allowed_stride, rows, vocab, _stream(dev))
    return logits
