"""MI355X HIP paged KV backend: fused decode attention, KV append and paged
prefill attention.

Drop-in for minivllm/triton_paged_decode.py. Inputs match
paged_attention_batch_online_v1:
    q:               [B, H, D] (arbitrary strides)
    pool.k / pool.v: [L, N, S, H, D]
    block_tables:    [B, M] (logical -> physical; -1 only in the unused tail)
    context_lengths: [B] (>= 1, include the KV written this step)

The entry points validate on the host exactly like
paged_attention_batch_triton_v0 (minivllm/triton_paged_decode.py:109-144):
ValueError for contract violations, RuntimeError when the HIP library or its
PyTorch binding is unavailable. The checks, allocations and launches run in
the binding (csrc/torch_ops.cpp), which calls the C ABI of
libminivllm_hip.so. Nothing reads device data on the host (no .item()); the
kernels launch on torch's current stream, so the KV append is ordered before
the attention that reads it. There is no fallback: without the library or a
GPU these functions raise.

Beyond the Triton v0 backend: float32, bfloat16 and float16; head_dim up to
512; any block size; a split of long and ragged contexts over many
wavefronts (all sequences' blocks dealt out evenly) with a merge pass.

paged_prefill_hip is the prefill counterpart (the reference's per-token
loop, minivllm/attention.py:269-299, and its sdpa_v2 gather,
minivllm/attention.py:229-267): causal attention of one chunk's queries over
the sequence's cached prefix and the chunk itself, read from the pool.

qk_norm_rope_hip and kv_append_rope_hip norm and rotate query and key heads by
their positions, the latter on the way into the pool.
paged_attention_shared_prefix_hip is decode attention, with grouped query
heads, for sequences that begin with the same cached blocks. kv_append_fp4,
kv_gather_fp4 and paged_attention_fp4_hip write, read back and attend over a
FP4KVBlockPool, whose keys and values are 4 bits. prompt_attention_hip is causal
attention of packed whole prompts over their own keys and values. These seven are
inference-only (RuntimeError for tensors that require gradients while grad mode
is on) and run on their tensors' device, current or not.
"""
from __future__ import annotations

import torch

from . import _native
from .kv_block_pool import FP4KVBlockPool, KVBlockPool


def paged_attention_batch_hip(q: torch.Tensor, pool: KVBlockPool, block_tables: torch.Tensor,
                              context_lengths: torch.Tensor, layer_idx: int, *,
                              split_tokens: int = 0) -> torch.Tensor:
    """One fused decode-attention pass over the paged pool; caller already wrote new KV.

    Returns a fresh [B, H, D] tensor of q.dtype. ``split_tokens`` = 0 lets
    the library split the work (evenly over a fixed number of wavefronts
    when contexts span several partitions); > 0 cuts every context into
    partitions of that many tokens.

    Validation (ValueError, the messages of the Triton v0 backend's checks),
    allocation and the launch happen in the _hip_ops binding
    (csrc/torch_ops.cpp).
    """
    return _native.ops().paged_decode(q, pool.k, pool.v, block_tables, context_lengths, int(layer_idx),
                                      int(split_tokens))


def paged_attention_batch_append_hip(q: torch.Tensor, pool: KVBlockPool, block_tables: torch.Tensor,
                                     context_lengths: torch.Tensor, layer_idx: int, k: torch.Tensor,
                                     v: torch.Tensor, slot_mapping: torch.Tensor, *,
                                     split_tokens: int = 0) -> torch.Tensor:
    """One decode step's KV write and attention as one call: kv_append of the
    B rows k[b], v[b] ([B, H, D]) into slot_mapping[b], then
    paged_attention_batch_hip, on the current stream.

    Where the library can (bf16/f16/f32 rows of the pool's dtype, head dim
    contiguous, 16-byte aligned, the fast attention path) the write runs inside
    the attention launch, by the wavefront that streams each sequence's last
    block, before it reads that block: one launch fewer per layer. The pool and
    the output are bit-identical to the two calls, given the decode step's
    invariant that a slot some context reads is the slot of its own row's last
    position (``context_lengths[b] - 1``); negative slots are skipped.
    """
    return _native.ops().paged_decode_append(q, pool.k, pool.v, block_tables, context_lengths, int(layer_idx),
                                             k, v, slot_mapping, int(split_tokens))


def paged_attention_shared_prefix_hip(q: torch.Tensor, pool: KVBlockPool, block_tables: torch.Tensor,
                                      context_lengths: torch.Tensor, layer_idx: int, *,
                                      shared_blocks: int) -> torch.Tensor:
    """paged_attention_batch_hip for sequences that begin with the same cached
    blocks: the first ``shared_blocks`` entries of every row of block_tables are
    taken from row 0 (the others' are not read), and those blocks' keys and
    values are read once for all rows, on the matrix cores; by each row itself in
    calls too small for that to pay, past 4096 rows, and where head_dim is over 256 or
    no multiple of 8 or rows are not contiguous and 16-byte aligned (the last by a slow
    kernel).

    q: [B, Hq, D] with Hq a multiple of the pool's heads H; query head h reads KV
    head h // (Hq // H). context_lengths count a sequence's tokens, the shared ones
    included; a sequence shorter than the shared blocks (a padding row of
    length 0, say) is attended by itself. shared_blocks = 0 is decode attention
    with grouped query heads. Returns a fresh [B, Hq, D] tensor of q.dtype. 2-byte
    types round the softmax weights to their type for the product with the values, as
    paged_prefill_hip does and paged_attention_batch_hip does not (bfloat16: 0.0023 off
    64 bits, relative, instead of 0.0017); sums are float32.
    """
    return _native.ops().paged_decode_shared(q, pool.k, pool.v, block_tables, context_lengths, int(layer_idx),
                                             int(shared_blocks))


def kv_append(pool: KVBlockPool, layer_idx: int, k: torch.Tensor, v: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
    """Scatters rows k[t], v[t] ([T, H, D], any strides) into pool slots slot_mapping[t].

    pool.k[layer, s // S, s % S] = k[t] (same for v) for every s >= 0; rows
    with a negative slot are skipped. Bit-exact when k/v share the pool dtype.
    """
    _native.ops().kv_append(pool.k, pool.v, int(layer_idx), k, v, slot_mapping)


def rope_table(positions: int, rotary_dim: int, *, base: float = 10000.0, device=None) -> torch.Tensor:
    """The cos_sin table of the rotary calls: [positions, rotary_dim] float32, row p
    holding the cosines of p * base ** (-2 i / rotary_dim), i < rotary_dim / 2, then
    the sines. The angles are computed in 64 bits, as 32 lose far positions."""
    if positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rope_table needs positions >= 1 and an even rotary_dim")
    half = rotary_dim // 2
    freq = base ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def qk_norm_rope_hip(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                     q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, *,
                     eps: float = 1e-6, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head (with the weights, [D]) and the
    rotation by its row's position, in one pass.

    q: [T, Hq, D], k: [T, Hk, D], any strides; positions: [T] integers; cos_sin: a
    rope_table of rotary_dim <= D. Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1)
    when ``interleaved``; dims past rotary_dim are normed only. Arithmetic is
    float32, rounded once. A position outside the table gives NaN in the rotated
    dims. Returns fresh contiguous (q_out, k_out).
    """
    return _native.ops().qk_norm_rope(q, k, positions, cos_sin, q_weight, k_weight, float(eps), bool(interleaved))


def kv_append_rope_hip(pool: KVBlockPool, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       slot_mapping: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                       q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, *,
                       eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """kv_append of the rotated keys and the values, and the rotated queries, in
    one launch: qk_norm_rope_hip's norms (with weights) and rotation, the keys
    and values written to the pool's slots under kv_append's rules.

    q: [T, Hq, D]; k, v: [T, H, D] of the pool's H heads; a chunk's T rows or a decode
    batch's. Returns the queries, [T, Hq, D] in the pool's dtype, for the attention
    that follows. Rows with a negative slot, or a position outside the table,
    leave the pool as it was. Of rows on one slot the last is kept, K and V both, in
    calls of up to 256 rows; in longer ones each element is one of theirs.
    """
    return _native.ops().kv_append_rope(pool.k, pool.v, int(layer_idx), q, k, v, slot_mapping, positions, cos_sin,
                                        q_weight, k_weight, float(eps), bool(interleaved))


def kv_append_fp4(pool: FP4KVBlockPool, layer_idx: int, k: torch.Tensor, v: torch.Tensor,
                  slot_mapping: torch.Tensor) -> None:
    """kv_append into a 4-bit pool: rows k[t], v[t] ([T, H, D], any strides; float32,
    bfloat16 or float16) are quantised (FP4KVBlockPool says how) on their way to slots
    slot_mapping[t]. Rows with a slot outside the pool are skipped; of rows on one slot
    the last is kept.
    """
    _native.ops().kv_append_fp4(pool.data, pool.block_size, pool.head_dim, int(layer_idx), k, v, slot_mapping)


def kv_gather_fp4(pool: FP4KVBlockPool, layer_idx: int, slot_mapping: torch.Tensor, *,
                  dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """The values slots slot_mapping[t] of a 4-bit pool hold: fresh (k, v), [T, H, D] of
    ``dtype`` (float32 and bfloat16 exactly; float16 as far as it reaches). Rows whose
    slot is outside the pool are 0.
    """
    return _native.ops().kv_gather_fp4(pool.data, pool.block_size, pool.head_dim, int(layer_idx), slot_mapping, dtype)


def paged_attention_fp4_hip(q: torch.Tensor, pool: FP4KVBlockPool, block_tables: torch.Tensor,
                            context_lengths: torch.Tensor, layer_idx: int) -> torch.Tensor:
    """paged_attention_batch_hip over the values a 4-bit pool holds, with grouped query
    heads: q is [B, Hq, D] with Hq a multiple of the pool's heads H, and query head h reads
    KV head h // (Hq // H). float32, bfloat16 or float16 queries; head_dim up to 256; any
    block size (16-token runs of a block are read fastest: a multiple of 16). Sums are
    float32 and the result is rounded once. Returns a fresh [B, Hq, D] tensor of q.dtype.
    """
    return _native.ops().paged_decode_fp4(q, pool.data, pool.block_size, pool.head_dim, block_tables,
                                          context_lengths, int(layer_idx))


def paged_prefill_hip(q: torch.Tensor, pool: KVBlockPool, block_table: torch.Tensor,
                      start_pos: int, layer_idx: int) -> torch.Tensor:
    """Causal attention of a chunk's queries through the paged pool.

    q: [T, H, D] (any strides), query row t at absolute position start_pos + t.
    block_table: [n] integer tensor of the sequence's physical blocks,
    n >= ceil((start_pos + T) / S). The chunk's own K/V must already be in
    the pool (kv_append on the same stream). Returns a fresh [T, H, D]
    tensor of q.dtype with out[t] = softmax(q[t] K[0..start_pos+t]^T / sqrt(D)) V.
    """
    return _native.ops().paged_prefill(q, pool.k, pool.v, block_table, int(start_pos), int(layer_idx))


def prompt_attention_hip(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor) -> torch.Tensor:
    """Causal attention of whole prompts, packed one after the other, over their own keys
    and values as the projection made them (no pool: append them to any pool beside it).

    q: [T, Hq, D]; k, v: [T, Hk, D] with Hq a multiple of Hk, any strides; query head h
    reads KV head h // (Hq // Hk). cu_seqlens: [B + 1] integers that never fall, sequence b
    being rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (none, for an empty one); it is read
    on the GPU alone, so a captured graph follows it. float32, bfloat16 or float16;
    head_dim up to 256. Returns a fresh [T, Hq, D] tensor of q.dtype; rows of no sequence
    are 0. A row's bits do not depend on rows it does not see, whatever they hold.
    """
    return _native.ops().prompt_attention(q, k, v, cu_seqlens)
