"""Functional wrappers over the sm_100a kernels.

Every function here launches kernels from ``kapsl_sdk_b200._cuda`` on the
current CUDA stream.  Plain fp32 PyTorch restatements of the same math live in
:mod:`kapsl_sdk_b200.ops.reference`; the CPU backend and the numerics tests use
them as the oracle.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from .._ext import cuda_ops

EPI_PLAIN, EPI_BIAS, EPI_RESIDUAL, EPI_SWIGLU = 0, 1, 2, 3

_err_bufs: dict[int, torch.Tensor] = {}


def error_buffer(device: torch.device) -> torch.Tensor:
    """Per-device int32[16] status words written by kernels whose bounded
    waits time out (0 = ok).  Read with :func:`check_errors`."""
    if device.type != "cuda":
        raise RuntimeError(f"the kernels take CUDA tensors, got one on {device}")
    idx = device.index if device.index is not None else torch.cuda.current_device()
    buf = _err_bufs.get(idx)
    if buf is None:
        buf = torch.zeros(16, dtype=torch.int32, device=device)
        _err_bufs[idx] = buf
    return buf


# Status codes the kernels record in the error buffer when a bounded wait runs out
# (or a size check fails); 0 = ok.
DEVICE_ERRORS = {
    1: "decode attention: a KV page load did not arrive within its wait limit",
    2: "prefill attention: a KV page load did not arrive within its wait limit",
    **{c: "GEMM pipeline wait ran out (1-SM kernel)" for c in range(10, 14)},
    **{c: "GEMM pipeline wait ran out (2-SM kernel)" for c in range(20, 24)},
    30: "tensor-parallel reduction (push): a peer missed barrier 1",
    31: "tensor-parallel reduction (push): a peer missed barrier 2",
    32: "tensor-parallel reduction (pull): a peer missed barrier 1",
    33: "tensor-parallel reduction (pull): a peer missed barrier 2",
    34: "tensor-parallel reduction + norm (pull): a peer missed barrier 1",
    35: "tensor-parallel reduction + norm (pull): a peer missed barrier 2",
    36: "tensor-parallel row reduction: a peer's partial rows did not arrive",
    37: "tensor-parallel row reduction: an owner's normed rows did not arrive",
    38: "tensor-parallel row reduction (LL): a peer's partial rows did not arrive",
    39: "NVLink flag probe: the peer's flag did not arrive",
    40: "MoE permute: expert rows exceed the sorted buffer",
    41: "MoE combine: a peer missed barrier 1",
    42: "MoE combine: a peer missed barrier 2",
    50: "vocab-parallel sampler: a peer's candidates did not arrive",
    **{c: "Q4_K GEMM pipeline wait ran out" for c in range(60, 67)},
    **{c: "tcgen05 prefill attention pipeline wait ran out" for c in range(71, 79)},
    80: "rotary positions: a position lies outside the cos/sin table (its row was not rotated)",
    81: "latent cache write: a slot lies outside the cache (its row was not written)",
    82: "latent attention: a block table entry lies outside the cache (its keys read as zeros)",
    83: "latent decode attention: shared memory is not 1 KiB aligned",
    **{c: "latent decode attention pipeline wait ran out" for c in range(84, 90)},
    90: "latent prefill attention: the plan's rows lie outside q, or shared memory is not 1 KiB aligned",
    **{c: "latent prefill attention pipeline wait ran out" for c in range(91, 97)},
    **{c: "latent expansion pipeline wait ran out" for c in range(97, 100)},
}


def describe_error(code: int) -> str:
    return f"device error {code}: {DEVICE_ERRORS.get(code, 'unknown status')}"


def check_errors(device: torch.device) -> int:
    """Return (and clear) the first non-zero kernel status word on ``device`` (0 for a device that
    runs no kernels)."""
    if device.type != "cuda":
        return 0
    buf = error_buffer(device)
    v = int(buf.max().item())
    if v:
        buf.zero_()
    return v


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out = rmsnorm(x [+ residual]) * weight``; with ``residual`` the sum is
    also stored back into ``residual`` (pre-norm residual stream update)."""
    if out is None:
        out = torch.empty_like(x)
    cuda_ops().rmsnorm(out, x, weight, float(eps), residual)
    return out


def rope_kv_write(qkv: torch.Tensor, positions: torch.Tensor, slots: Optional[torch.Tensor], cos_sin: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, num_heads: int, num_kv_heads: int,
                  head_dim: int) -> None:
    """Rotate q and k of ``qkv`` in place and write k, v into the paged cache."""
    cuda_ops().rope_kv_write(qkv, positions, slots, cos_sin, k_cache, v_cache, num_heads, num_kv_heads, head_dim)


def rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, offset: int = 0, interleaved: bool = False,
         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions of the heads of ``x`` [T, H, D] (bf16, fp16 or fp32; any token and head
    strides): the dims ``[offset, offset + P)`` of every head turn by their token's angles,
    the others are copied.  ``cos_sin`` [positions, P] comes from
    :func:`~kapsl_sdk_b200.ops.reference.rope_cos_sin` (scaled tables included), so its
    width is the rotated part.  Pairs are ``(i, i + P/2)``, or ``(2i, 2i + 1)`` with
    ``interleaved``.  ``out=x`` rotates in place.  A position outside the table leaves its
    row unrotated and records device error 80."""
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    cuda_ops().rope(out, x, positions, cos_sin, int(offset), bool(interleaved), error_buffer(x.device))
    return out


def rope_latent_write(q_rope: torch.Tensor, kv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                      cos_sin: torch.Tensor, weight: torch.Tensor, eps: float, cache: torch.Tensor,
                      interleaved: bool = False, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step's cache write of latent attention, with the queries' rotation.

    ``kv`` [T, R + 64] (R 256 or 512) is a token's compressed row: the first R values are RMS-normed
    with ``weight``, the last 64 rotated by ``positions``, and the row goes to
    ``cache`` [blocks, page, R + 64] at ``slots[t]`` = block * page + offset (a negative slot marks
    a padded row: nothing is written, and its position is not looked at for errors; a slot past
    the cache is skipped and records device error 81).  A position outside the table leaves its
    key and queries unrotated and, unless the row is padded, records device error 80.
    ``q_rope`` [T, H, 64], the rotary part of the query heads (usually a view
    ``q.view(T, H, 192)[..., 128:]``), is rotated in place, or into ``q_out``.
    Two tokens of one call must not share a slot."""
    if q_out is None:
        q_out = q_rope
    cuda_ops().rope_latent_write(q_rope, q_out, kv, positions, slots, cos_sin, weight, float(eps), cache,
                                 bool(interleaved), error_buffer(q_rope.device))
    return q_out


def silu_mul(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    F = x.shape[1] // 2
    if out is None:
        out = torch.empty(x.shape[0], F, dtype=x.dtype, device=x.device)
    cuda_ops().silu_mul(out, x)
    return out


def embedding(ids: torch.Tensor, table: torch.Tensor, vocab_start: int = 0,
              out: Optional[torch.Tensor] = None, src_rows: Optional[torch.Tensor] = None,
              prev_tokens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of ``table`` for ``ids``.  With ``src_rows``: row ``t < len(src_rows)``
    whose ``src_rows[t] >= 0`` looks up ``prev_tokens[src_rows[t]]`` instead of
    ``ids[t]`` (a token the previous step sampled and the host has not read yet)."""
    if out is None:
        out = torch.empty(ids.numel(), table.shape[1], dtype=table.dtype, device=table.device)
    cuda_ops().embedding(out, table, ids, int(vocab_start), src_rows, prev_tokens)
    return out


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, swiglu: bool = False, out: Optional[torch.Tensor] = None,
           out_dtype: torch.dtype = torch.bfloat16, workspace: Optional[torch.Tensor] = None,
           force_bn: int = 0, force_splits: int = 0) -> torch.Tensor:
    """``out = epilogue(x @ weight.T)`` on the tcgen05 GEMM.

    Exactly one of ``bias`` / ``residual`` / ``swiglu`` selects the fused
    epilogue.  ``residual`` may be the same tensor as ``out`` (in-place
    residual-stream update).  ``swiglu`` expects the gate/up weight interleaved
    in 128-row blocks (see :func:`interleave_gate_up`) and returns [M, N/2].
    """
    if not isinstance(weight, torch.Tensor):
        return _quant_linear(x, weight, bias, residual, swiglu, out, out_dtype, workspace)
    M, N = x.shape[0], weight.shape[0]
    epi = EPI_PLAIN
    if bias is not None:
        epi = EPI_BIAS
    elif residual is not None:
        epi = EPI_RESIDUAL
    elif swiglu:
        epi = EPI_SWIGLU
    ncols = N // 2 if swiglu else N
    if out is None:
        out = torch.empty(M, ncols, dtype=out_dtype, device=x.device)
    if workspace is None:
        workspace = _workspace(x.device)
    cuda_ops().gemm(x, weight, out, epi, bias, residual, workspace, error_buffer(x.device), force_bn, force_splits)
    return out


# Token count and weight rows from which a Q4_K product dequantizes the whole weight
# matrix to bf16 (one memory-bound pass, ~20.5 bits moved per weight) and runs the
# bf16 tcgen05 GEMM, instead of the fused kernel that dequantizes each weight tile
# again for every 256-token tile.  Measured on B200 (ms, fused -> dequant + bf16):
# 2048 x 8192 x 3584 0.135 -> 0.112, 2048 x 57344 x 8192 1.99 -> 1.69, 2048 x 7168 x 8192
# 0.242 -> 0.231; the fused kernel stays ahead at 1024 tokens (0.126 vs 0.143) and on
# narrow products (2048 x 1280 x 8192: 0.067 vs 0.100).
Q4K_DEQUANT_MIN_M = 2048
Q4K_DEQUANT_MIN_N = 4096

_q4k_scratch: dict[int, torch.Tensor] = {}


def _q4k_weight_scratch(device: torch.device, numel: int) -> Optional[torch.Tensor]:
    """Per-device bf16 buffer for a dequantized weight matrix, grown on demand;
    None when it would have to grow while a CUDA graph is being captured."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    buf = _q4k_scratch.get(idx)
    if buf is None or buf.numel() < numel:
        if torch.cuda.is_current_stream_capturing():
            return None
        buf = torch.empty(numel, dtype=torch.bfloat16, device=device)
        _q4k_scratch[idx] = buf
    return buf


def _quant_linear(x, weight, bias, residual, swiglu, out, out_dtype, workspace) -> torch.Tensor:
    """``linear`` for a :class:`~kapsl_sdk_b200.quantization.QuantWeight` (Q4_K):
    the fused dequant GEMM, with residual fused; SwiGLU expects the gate and up
    rows concatenated ([gate; up], not interleaved).  From ``Q4K_DEQUANT_MIN_M``
    tokens and ``Q4K_DEQUANT_MIN_N`` weight rows the weight is dequantized into a scratch matrix (gate/up rows written
    in the interleaved SwiGLU layout) and the bf16 GEMM runs with the same
    epilogue."""
    if weight.fmt != "q4_k":
        raise ValueError(f"no fused kernel for weight format {weight.fmt!r}")
    if out_dtype != torch.bfloat16:
        raise ValueError("quantized linear layers produce bf16")
    M, N = x.shape[0], weight.n
    if workspace is None:
        workspace = _workspace(x.device)
    c = cuda_ops()
    err = error_buffer(x.device)
    if M >= Q4K_DEQUANT_MIN_M and N >= Q4K_DEQUANT_MIN_N and (not weight.tiled or N % 128 == 0):
        buf = _q4k_weight_scratch(x.device, N * weight.k)
        if buf is not None:
            w = buf[:N * weight.k].view(N, weight.k)
            half = N // 2 if swiglu and N % 256 == 0 else 0
            c.q4k_dequant_rows(weight.raw, N, weight.k, weight.tiled, half, w)
            if swiglu and half:
                return linear(x, w, swiglu=True, out=out, workspace=workspace)
            if swiglu:
                return silu_mul(linear(x, w, workspace=workspace), out)
            y = linear(x, w, residual=residual, out=out, workspace=workspace)
            if bias is not None:
                y.add_(bias)
            return y
    if swiglu:
        y = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
        c.gemm_q4k(x, weight.raw, y, weight.k, None, workspace, 0, weight.tiled, err)
        return silu_mul(y, out)
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    c.gemm_q4k(x, weight.raw, out, weight.k, residual, workspace, 0, weight.tiled, err)
    if bias is not None:
        out.add_(bias)
    return out


_ws: dict[int, torch.Tensor] = {}


def _workspace(device: torch.device, nbytes: int = 64 << 20) -> torch.Tensor:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _ws.get(idx)
    if w is None or w.numel() * 4 < nbytes:
        w = torch.empty(nbytes // 4, dtype=torch.float32, device=device)
        _ws[idx] = w
    return w


def workspace(device: torch.device) -> torch.Tensor:
    """The per-device fp32 GEMM workspace (split-K partials)."""
    return _workspace(device)


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor, block: int = 128) -> torch.Tensor:
    """[F, d] gate and up -> [2F, d] with alternating 128-row blocks
    (gate_0, up_0, gate_1, up_1, ...), the layout the SwiGLU epilogue reads."""
    F, d = gate.shape
    assert F % block == 0, "intermediate size must be a multiple of 128"
    g = gate.view(F // block, block, d)
    u = up.view(F // block, block, d)
    return torch.stack([g, u], dim=1).reshape(2 * F, d).contiguous()


def decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                     ctx_lens: torch.Tensor, num_heads: int, num_kv_heads: int, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, num_splits: int = 0,
                     scratch: Optional[tuple[torch.Tensor, torch.Tensor]] = None,
                     max_ctx: Optional[int] = None) -> torch.Tensor:
    """Paged decode attention (one query token per row of ``q``)."""
    B = q.shape[0]
    D = 128
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty(B, num_heads * D, dtype=q.dtype, device=q.device)
    ops = cuda_ops()
    if num_splits <= 0:
        mc = int(max_ctx) if max_ctx is not None else int(block_tables.shape[1]) * 16
        num_splits = int(ops.decode_num_splits(B, num_kv_heads, mc))
    po = pl = None
    if num_splits > 1:
        if scratch is None:
            po = torch.empty(B * num_heads * num_splits * D, dtype=torch.float32, device=q.device)
            pl = torch.empty(B * num_heads * num_splits, dtype=torch.float32, device=q.device)
        else:
            po, pl = scratch
    ops.decode_attention(q, k_cache, v_cache, block_tables, ctx_lens, out, num_heads, num_kv_heads, float(scale),
                         num_splits, po, pl, error_buffer(q.device))
    return out


def prefill_work(q_lens: list[int], tile: int = 64) -> list[tuple[int, int]]:
    """Work list of (sequence, first query row) tiles for :func:`prefill_attention`."""
    work = []
    for s, n in enumerate(q_lens):
        for t0 in range(0, n, tile):
            work.append((s, t0))
    return work


def prefill_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, work: torch.Tensor,
                      seq_info: torch.Tensor, block_tables: torch.Tensor, num_heads: int, num_kv_heads: int,
                      out: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Chunked-prefill attention.  ``seq_info[s] = (q_start, q_len, ctx_len, bt_row)``;
    the chunk's tokens sit at positions ``ctx_len - q_len .. ctx_len - 1``."""
    if scale is None:
        scale = 1.0 / math.sqrt(128)
    cuda_ops().prefill_attention(q, k_cache, v_cache, work, seq_info, block_tables, out, num_heads, num_kv_heads,
                                 float(scale), error_buffer(q.device))
    return out


def prefill_attention_tc(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, work: torch.Tensor,
                         seq_info: torch.Tensor, block_tables: torch.Tensor, num_heads: int, num_kv_heads: int,
                         out: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """:func:`prefill_attention` on the tcgen05 kernel; ``work`` from
    ``prefill_work(q_lens, tile=prefill_tc_tile(num_heads, num_kv_heads))``."""
    if scale is None:
        scale = 1.0 / math.sqrt(128)
    cuda_ops().prefill_attention_tc(q, k_cache, v_cache, work, seq_info, block_tables, out, num_heads, num_kv_heads,
                                    float(scale), error_buffer(q.device))
    return out


def prefill_tc_tile(num_heads: int, num_kv_heads: int) -> int:
    """Query tokens per CTA of the tcgen05 prefill kernel: its 128 MMA rows hold
    every query head of one KV head for floor(128 / group) tokens."""
    return 128 // (num_heads // num_kv_heads)


# ------------------------------------------------------------ latent attention
def latent_decode_attention(q: torch.Tensor, cache: torch.Tensor, w_kv_b: torch.Tensor, block_tables: torch.Tensor,
                            ctx_lens: torch.Tensor, num_heads: int, scale: Optional[float] = None,
                            out: Optional[torch.Tensor] = None, max_ctx: Optional[int] = None) -> torch.Tensor:
    """Latent attention of one query token per row, absorbed form.

    ``cache`` [blocks, page, R + 64] holds one row a token (:func:`rope_latent_write`; R 256 or
    512, pages of 16, 32 or 64).  ``w_kv_b`` [H * 256, R] expands a latent to every head's
    128 key and 128 value dims; here its key half moves to the query's side and its value
    half is applied to the attended latents, so nothing is expanded per cached token.
    ``q`` [B, H * 192] has 128 position-free and 64 rotated dims a head; ``out`` is
    [B, H * 128].  Rows with ``ctx_lens`` 0 (a padded batch) and rows whose scores are all -inf give
    zeros; a context longer than its block table is cut to the table.  ``max_ctx`` (a host number,
    default the block tables' width) only bounds how many CTAs are launched.
    The keys of a block table entry outside the cache read as zeros, and device error 82 is recorded."""
    if scale is None:
        scale = 1.0 / math.sqrt(192)
    if out is None:
        out = torch.empty(q.shape[0], num_heads * 128, dtype=q.dtype, device=q.device)
    if max_ctx is None:
        max_ctx = block_tables.shape[-1] * cache.shape[1]
    c = cuda_ops()
    ws = torch.empty(c.latent_workspace_bytes(q, num_heads, cache.shape[-1] - 64, max_ctx), dtype=torch.uint8,
                     device=q.device)
    c.latent_decode_attention(q, cache, w_kv_b, block_tables, ctx_lens, out, num_heads, float(scale), max_ctx, ws,
                              None, error_buffer(q.device))
    return out


LATENT_PREFILL_TILE = 256  # query tokens a CTA of the expanded-form attention handles
LATENT_KV_BYTES = 2 << 30  # expanded keys, values and partial results held at once; more heads go in further passes
LATENT_PART_BYTES = LATENT_PREFILL_TILE * 130 * 4  # partial result of one part of a row tile's keys and one head


@dataclass
class LatentPrefillPlan:
    """Tile list and sequence table of one :func:`latent_prefill_attention` call."""
    work: torch.Tensor      # int32 [n, 2]: (sequence, first new token) of every tile of query rows
    kv_work: torch.Tensor   # int32 [m, 2]: (sequence, first context row) of every 128 context rows
    seq_info: torch.Tensor  # int32 [S, 5]: (first q row, tokens, context, block-table row, first kv row)
    rows: int               # q rows up to the last sequence's end
    tables: int             # block-table rows read
    max_ctx: int
    kv_rows: int            # context rows of all sequences, each padded to a multiple of 16
    q_start: int
    row_ctx: torch.Tensor   # int32 [rows - q_start]: context of every new token (itself included)
    row_table: torch.Tensor  # int32 [rows - q_start]: its block-table row
    single_tiles: int       # 64-key tiles of all new tokens taken one by one
    row_tiles: int          # 128-key tiles of all 256-row tiles of new tokens
    chain_us: float         # the longest of those row tiles by itself (microseconds)
    key_tiles: list[int]    # 128-key tiles of each row tile, in the order of work (most first)

    def key_ranges(self, num_heads: int) -> int:
        """Parts into which the expanded form cuts the longest row tile's keys: as often as it takes by
        itself what all row tiles take spread over the 148 SMs, parts of 4 key tiles or more.  512
        new tokens over 16384, 20 heads: 331 us whole, 188 in three parts; row tiles that fill the
        GPU stay whole, since parts cost fp32 partial results and a joining kernel."""
        spread = max(4.0, 1.9 * self.row_tiles * num_heads / 148)
        return max(1, min(32, -(-self.max_ctx // 128) // 4, int(self.chain_us / spread)))

    def passes(self, num_heads: int, key_ranges: int = 0) -> tuple[int, int, int, int]:
        """The expanded form's (heads a pass, row tiles cut, key tiles a part, parts of the longest row tile)
        under LATENT_KV_BYTES (one head may take more keys and values than that).  Only row tiles longer
        than a part are cut: the others write no partial results.  One chunk of 256 tokens over 65,536 beside
        500 single tokens, 8 heads: 10 MB of them for one row tile; cutting all 501 took 4.8 GB."""
        kv = max(1, self.kv_rows * 512)
        step = max(1, min(num_heads, LATENT_KV_BYTES // kv))
        ranges = key_ranges if key_ranges > 0 else self.key_ranges(step)
        while ranges > 1 and self.key_tiles:
            part = -(-self.key_tiles[0] // ranges)
            cut, slots = sum(n > part for n in self.key_tiles), -(-self.key_tiles[0] // part)
            room = cut * slots * LATENT_PART_BYTES
            if room <= LATENT_KV_BYTES:
                return max(1, min(step, LATENT_KV_BYTES // (kv + room))), cut, part, slots
            ranges //= 2
        return step, 0, 0, 1

    def absorbed_is_shorter(self, num_heads: int, rank: int = 512) -> bool:
        """Whether taking every new token by itself in the absorbed form is estimated to take less time
        than expanding the contexts.  In microseconds, fitted to both forms' times on a B200's 148
        SMs over some 40 ragged batches: absorbed, a 64-key tile of up to 64 heads 3.0 (rank 256:
        1.4) of an SM, of 65 - 128 heads 2.6 (rank 256: 2.8), and 2 for a thousand rows x heads of
        head products; expanded, 256 context rows of a head 4.5 (2.3) of an SM pair, a 128-key tile
        of 256 new tokens 1.9 of an SM, or the longest row tile by itself, or a part of it and 9 for
        the join.  20 new tokens over 4020, 8 heads: 37 and 46; five prompts of 17 to 300 tokens, 28
        heads: 98 and 59.  Small absorbed calls of more than 64 heads take up to 1.5 times the
        estimate (45 us for 30), where the choice was still right to a few percent.  One choice is made
        for the whole call: a few tokens over a long context beside a long prompt take its form."""
        rows, wide, ranges = self.rows - self.q_start, rank > 256, self.key_ranges(num_heads)
        start = 19 if -(-rows // 16) * num_heads <= 256 else 26
        tile = (2.6 * -(-num_heads // 128) if wide and num_heads > 64 else
                (3.0 if wide else 1.4) * -(-num_heads // 64))
        absorbed = start + tile * self.single_tiles / 148 + 0.002 * rows * num_heads
        expanded = 20 + 1.2 * ((4.5 if wide else 2.3) * -(-self.kv_work.shape[0] // 2) * num_heads / 74 +
                               max(self.chain_us / ranges, 1.9 * self.row_tiles * num_heads / 148) +
                               9 * (ranges > 1))
        return absorbed < expanded and rows <= 4096


def latent_prefill_plan(q_lens: Sequence[int], ctx_lens: Sequence[int], device, q_start: int = 0,
                        bt_start: int = 0) -> LatentPrefillPlan:
    """Plan of chunks of ``q_lens[s]`` new tokens at the end of contexts of ``ctx_lens[s]`` tokens
    (new ones included).  Their q rows follow each other from ``q_start``, their block
    tables from row ``bt_start`` (a mixed batch has its decode rows first).  The tables are
    device tensors: reuse them for every layer of a step."""
    q_lens, ctx_lens = [int(n) for n in q_lens], [int(n) for n in ctx_lens]
    if len(q_lens) != len(ctx_lens):
        raise ValueError("latent_prefill_plan: q_lens and ctx_lens differ in length")
    if q_start < 0 or bt_start < 0:
        raise ValueError("latent_prefill_plan: negative start")
    info, work, row, kv = [], [], int(q_start), 0
    row_ctx, row_table, single, chain = [], [], 0, 0.0

    def tiles64(c: int) -> int:  # 64-key tiles of contexts 1 .. c, summed
        full = c // 64
        return 32 * full * (full + 1) + (c % 64) * (full + 1)

    for s, (n, ctx) in enumerate(zip(q_lens, ctx_lens)):
        if n < 0 or n > ctx:
            raise ValueError(f"latent_prefill_plan: sequence {s} has {n} new tokens in a context of {ctx}")
        if n == 0:  # nothing asks for its context
            ctx = 0
        info.append((row, n, ctx, bt_start + s, kv))
        for t0 in range(0, n, LATENT_PREFILL_TILE):
            keys = ctx - n + min(n, t0 + LATENT_PREFILL_TILE)
            work.append((keys, s, t0))
            chain = max(chain, -(-keys // 128) * (1.35 if n - t0 <= 128 else 1.9))
        row_ctx.append(torch.arange(ctx - n + 1, ctx + 1, dtype=torch.int32))
        row_table.append(torch.full((n,), bt_start + s, dtype=torch.int32))
        single += tiles64(ctx) - tiles64(ctx - n)
        row += n
        kv += -(-ctx // 16) * 16
    if row >= 2 ** 31 or kv >= 2 ** 31:
        raise ValueError("latent_prefill_plan: too many rows")
    work.sort(key=lambda w: -w[0])  # the tiles with the most keys start first
    dev = torch.device(device)
    kv_work = [(s, r) for s, i in enumerate(info) for r in range(0, i[2], 128)]
    parts = [torch.tensor(v, dtype=torch.int32) for v in (
        [v for w in work for v in w[1:]], [v for w in kv_work for v in w], [v for i in info for v in i])]
    none = torch.empty(0, dtype=torch.int32)
    parts += [torch.cat(row_ctx or [none]), torch.cat(row_table or [none])]
    t = torch.cat(parts).to(dev).split([p.numel() for p in parts])
    return LatentPrefillPlan(work=t[0].view(-1, 2), kv_work=t[1].view(-1, 2), seq_info=t[2].view(-1, 5), rows=row,
                             tables=bt_start + len(info) if info else 0, max_ctx=max([i[2] for i in info], default=0),
                             kv_rows=kv, q_start=int(q_start), row_ctx=t[3], row_table=t[4], single_tiles=single,
                             row_tiles=sum(-(-w[0] // 128) for w in work), chain_us=chain,
                             key_tiles=[-(-w[0] // 128) for w in work])


def latent_prefill_attention(q: torch.Tensor, cache: torch.Tensor, w_kv_b: torch.Tensor, plan: LatentPrefillPlan,
                             block_tables: torch.Tensor, num_heads: int, scale: Optional[float] = None,
                             out: Optional[torch.Tensor] = None, form: Optional[str] = None,
                             key_ranges: int = 0) -> torch.Tensor:
    """Causal latent attention of chunks of new tokens over the paged latent cache.

    The new tokens' rows are in ``cache`` already; arguments as in
    :func:`latent_decode_attention`, with ``plan`` from :func:`latent_prefill_plan`.  In the
    expanded form the context's latents are expanded out of their pages by ``w_kv_b`` to keys
    and values (with partial results at most ``LATENT_KV_BYTES`` at a time, in passes over the heads); in
    the absorbed form every new token is a row of :func:`latent_decode_attention`, which is
    shorter for few of them.  ``form`` ("expanded" or "absorbed") overrides
    :meth:`LatentPrefillPlan.absorbed_is_shorter`, ``key_ranges`` (1 to 32, expanded form)
    :meth:`LatentPrefillPlan.key_ranges`; the two forms round differently.  Page slots behind
    a context may hold anything; its own latents have to be finite, since in the expanded form
    a row that is not also reaches earlier new tokens (0 * NaN in the product with the values).
    Rows whose scores are all -inf give zeros.  ``out`` rows outside the plan's sequences keep
    what they held (zeros when ``out`` is allocated here)."""
    if scale is None:
        scale = 1.0 / math.sqrt(192)
    if out is None:
        out = torch.zeros(q.shape[0], num_heads * 128, dtype=q.dtype, device=q.device)
    c = cuda_ops()
    c.check_latent_prefill(q, cache, w_kv_b, block_tables, out, num_heads, plan.rows, plan.tables, plan.max_ctx)
    if plan.work.shape[0] == 0:
        return out
    err = error_buffer(q.device)
    if form not in (None, "expanded", "absorbed"):
        raise ValueError(f"latent_prefill_attention: form {form!r}")
    if form == "absorbed" or (form is None and plan.absorbed_is_shorter(num_heads, cache.shape[2] - 64)):
        rows = slice(plan.q_start, plan.rows)
        ws = torch.empty(c.latent_workspace_bytes(q[rows], num_heads, cache.shape[2] - 64, plan.max_ctx),
                         dtype=torch.uint8, device=q.device)
        c.latent_decode_attention(q[rows], cache, w_kv_b, block_tables, plan.row_ctx, out[rows], num_heads,
                                  float(scale), plan.max_ctx, ws, plan.row_table, err)
        return out
    if key_ranges > 32:
        raise RuntimeError("latent_prefill_attention: 1 to 32 key ranges")
    w = w_kv_b.view(num_heads * 256, -1)
    step, cut, part, slots = plan.passes(num_heads, key_ranges)
    k_rope = torch.empty(plan.kv_rows, 64, dtype=torch.bfloat16, device=q.device)
    kv_buf = torch.empty(plan.kv_rows * step * 256, dtype=torch.bfloat16, device=q.device)
    parts = None
    if cut > 0:
        parts = torch.empty(cut * slots * step * LATENT_PART_BYTES // 4, dtype=torch.float32, device=q.device)
    for h0 in range(0, num_heads, step):
        n = min(step, num_heads - h0)
        kv = kv_buf[:plan.kv_rows * n * 256].view(plan.kv_rows, n * 256)
        c.latent_expand(cache, w[h0 * 256:(h0 + n) * 256], plan.kv_work, plan.seq_info, block_tables, kv,
                        k_rope if h0 == 0 else None, err)
        c.latent_prefill(q[:, h0 * 192:(h0 + n) * 192], kv, k_rope, plan.work, plan.seq_info,
                         out[:, h0 * 128:(h0 + n) * 128], n, float(scale), cut, part, slots, parts, err)
    return out


SAMPLE_MAX_TOP_K = 1024  # top_k above this (or 0, with T > 0) takes the whole-vocabulary path


def sample(logits: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor, top_p: torch.Tensor,
           rng_state: torch.Tensor, out: torch.Tensor, rep_penalty: Optional[torch.Tensor] = None,
           counts: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
           occ: Optional[torch.Tensor] = None, occ_n: Optional[torch.Tensor] = None,
           full_scratch: Optional[torch.Tensor] = None, full_ctas: int = 0) -> torch.Tensor:
    """Sample one token per row of fp32 ``logits`` (modified in place).

    ``rng_state`` (int64 LCG states), ``counts`` (per-id occurrence counts for
    the repetition penalty) and ``occ`` / ``occ_n`` (each slot's list of ids
    that occurred, so the penalty touches only those logits) are per-sequence
    tables indexed by ``slots[row]`` (or by the row itself when ``slots`` is
    None).  Rows with T > 0 and top_k 0 or > 1024 are sampled over the whole
    vocabulary when ``full_scratch`` (:func:`sample_full_scratch`) is given."""
    cuda_ops().sample(logits, temperature, top_k, top_p, rep_penalty, counts, slots, rng_state, out, occ, occ_n, 0,
                      logits.shape[1], full_scratch, int(full_ctas), [], [], 0, 0, None, 0,
                      error_buffer(logits.device))
    return out


def sample_full_scratch(vocab: int, device, ctas: int = 32) -> torch.Tensor:
    """Scratch for ``ctas`` rows sampled over the whole vocabulary at once."""
    n = int(cuda_ops().sample_full_scratch_bytes(vocab, ctas))
    return torch.empty(n, dtype=torch.uint8, device=device)


def count_tokens(counts: torch.Tensor, rows: torch.Tensor, ids: torch.Tensor, occ: Optional[torch.Tensor] = None,
                 occ_n: Optional[torch.Tensor] = None) -> None:
    """``counts[rows[i], ids[i]] += 1``; a first occurrence also appends the id to
    ``occ[rows[i]]`` (length ``occ_n[rows[i]]``)."""
    cuda_ops().count_tokens(counts, rows, ids, occ, occ_n)


# ------------------------------------------------------------ mixture of experts
def moe_route(x: torch.Tensor, w_router: torch.Tensor, top_k: int, renormalize: bool = True,
              ids: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None):
    """Router logits ``x @ w_router.T`` -> (expert ids int32 [T, k], weights fp32 [T, k])."""
    T = x.shape[0]
    if ids is None:
        ids = torch.empty(T, top_k, dtype=torch.int32, device=x.device)
    if weights is None:
        weights = torch.empty(T, top_k, dtype=torch.float32, device=x.device)
    cuda_ops().moe_route(x, w_router, top_k, renormalize, ids, weights)
    return ids, weights


def moe_permute(ids: torch.Tensor, num_experts: int, e_lo: int, e_local: int, max_rows: int, seg: torch.Tensor,
                pos: torch.Tensor, mtiles: torch.Tensor, src: torch.Tensor) -> None:
    """Stable expert sort of the [T, k] assignments (segments padded to 128 rows)."""
    T, k = ids.shape
    cuda_ops().moe_permute(ids, T, k, num_experts, e_lo, e_local, max_rows, seg, pos, mtiles, src,
                           error_buffer(ids.device))


def moe_gather(x: torch.Tensor, src: torch.Tensor, mtiles: torch.Tensor, xs: torch.Tensor) -> None:
    cuda_ops().moe_gather(x, src, mtiles, xs)


def grouped_linear(xs: torch.Tensor, w: torch.Tensor, n_per_group: int, mtiles: torch.Tensor,
                   out: torch.Tensor, swiglu: bool = False, splits: int = 1, bn: int = 0,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-expert GEMM over expert-sorted rows: tile i of ``xs`` times expert
    ``mtiles[1 + i]`` of ``w`` ([groups * n_per_group, K])."""
    groups = w.shape[0] // n_per_group
    if splits > 1 and workspace is None:
        workspace = _workspace(xs.device, splits * xs.shape[0] * n_per_group * 4)
    cuda_ops().grouped_gemm(xs, w, out, n_per_group, groups, mtiles, 3 if swiglu else 0, bn, splits, workspace,
                            error_buffer(xs.device))
    return out


def moe_combine(y_ptrs: list[int], hidden_ptrs: list[int], flag_ptrs: list[int], rank: int, ids: torch.Tensor,
                weights: torch.Tensor, pos: torch.Tensor, seg: torch.Tensor, e_local: int, cols: int, ld_y: int,
                ld_h: int, rows_per_rank: int, epoch: Optional[torch.Tensor] = None,
                timeout_ns: int = 5_000_000_000) -> None:
    """Weighted top-k combine + residual; with peers (len(y_ptrs) > 1) each wait on
    a peer's flag gives up after ``timeout_ns`` and records error 41 / 42."""
    T, k = ids.shape
    cuda_ops().moe_combine(y_ptrs, hidden_ptrs, flag_ptrs, rank, ids, weights, pos, seg, T, k, e_local, cols, ld_y,
                           ld_h, rows_per_rank, epoch, error_buffer(ids.device), int(timeout_ns))
