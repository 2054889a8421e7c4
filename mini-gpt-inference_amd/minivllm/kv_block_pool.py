"""Physical paged KV storage.

API of minivllm/kv_block_pool.py:32-152 (KVBlockPool): two tensors ``k`` and
``v`` of shape [n_layer, num_blocks, block_size, n_head, head_dim], created
with ``torch.empty`` (contents start undefined, so every reader must mask
slots past a sequence's length). Element strides are therefore
(N*S*H*D, S*H*D, H*D, D, 1): one physical block of one layer is a
contiguous [S, H, D] slab, and one token of one layer is a contiguous [H, D]
row -- the layout the HIP kernels read in place.
"""
from __future__ import annotations

import torch

from .sequence import SequenceState


def make_kv(seq_tag: int, logical_pos: int, n_layer: int, n_head: int, head_dim: int):
    """Deterministic per-(sequence, position) K/V of shape [n_layer, n_head, head_dim].

    Same values as minivllm/kv_block_pool.py:5-29: an arange pattern offset by
    ``seq_tag * 10000 + logical_pos * 100`` (V is K + 0.5).
    """
    base = torch.arange(n_layer * n_head * head_dim, dtype=torch.float32)
    base = base.reshape(n_layer, n_head, head_dim)
    shift = seq_tag * 10000 + logical_pos * 100
    return base + shift, base + (shift + 0.5)


class KVBlockPool:
    def __init__(self, n_layer: int, num_blocks: int, block_size: int, n_head: int,
                 head_dim: int, device="cpu", dtype=torch.float32):
        self.n_layer = n_layer
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.n_head = n_head
        self.head_dim = head_dim
        self.dtype = dtype
        shape = (n_layer, num_blocks, block_size, n_head, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)

    @property
    def device(self) -> torch.device:
        return self.k.device

    def write(self, physical_block: int, block_offset: int, k_new: torch.Tensor,
              v_new: torch.Tensor) -> None:
        """Writes one token slot in every layer; k_new/v_new are [L, H, D]."""
        expected = (self.n_layer, self.n_head, self.head_dim)
        assert tuple(k_new.shape) == expected
        assert tuple(v_new.shape) == expected
        self.k[:, physical_block, block_offset].copy_(k_new)
        self.v[:, physical_block, block_offset].copy_(v_new)

    def write_layer(self, layer_idx: int, physical_block: int, block_offset: int,
                    k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Writes one token slot of one layer; k_new/v_new are [H, D]."""
        self.k[layer_idx, physical_block, block_offset].copy_(k_new)
        self.v[layer_idx, physical_block, block_offset].copy_(v_new)

    def gather_sequence(self, seq: SequenceState) -> tuple[torch.Tensor, torch.Tensor]:
        """Logical K/V of `seq` on the host: two [L, seq.length, H, D] tensors."""
        length = seq.length
        S = self.block_size
        k_out = torch.empty((self.n_layer, length, self.n_head, self.head_dim), dtype=self.dtype)
        v_out = torch.empty_like(k_out)
        for logical, physical in enumerate(seq.block_table):
            lo = logical * S
            hi = min(lo + S, length)
            if hi <= lo:
                break
            k_out[:, lo:hi].copy_(self.k[:, physical, : hi - lo])
            v_out[:, lo:hi].copy_(self.v[:, physical, : hi - lo])
        return k_out, v_out


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_E2M1_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


class FP4KVBlockPool:
    """Paged KV storage in 4 bits, 17/64 of a bfloat16 pool's bytes.

    A head's row of head_dim elements (at most 256) is held in groups of 32 (the last
    padded with zeros): e2m1 values {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign, times one
    power of two per group, as the OCP microscaling formats have them. The scale is the
    least 2**e (-125 <= e <= 125) with max |x| <= 7 * 2**e and each element becomes the
    nearest value, ties to the even code, so it is off by at most 2**e. A group with an
    infinity or a NaN is held as NaN.

    ``data`` is [n_layer, num_blocks, n_head, slab] uint8. A slab is one block of one
    head: K codes [S, g * 16] (two to a byte, the even dim low), V codes [S, g * 16], K
    scales [S, g], V scales [g, S] (the byte is e + 127; 255 is NaN), with
    g = ceil(head_dim / 32), padded to 16 bytes. It is created with ``torch.empty``, as
    KVBlockPool is. write, write_layer and gather_sequence are KVBlockPool's (in PyTorch,
    on any device; one layer's rows at GPU speed: hip_paged_decode.kv_append_fp4).
    """

    GROUP = 32
    MAX_HEAD_DIM = 256

    def __init__(self, n_layer: int, num_blocks: int, block_size: int, n_head: int, head_dim: int, device="cpu"):
        if not 1 <= head_dim <= self.MAX_HEAD_DIM:
            raise ValueError("4-bit KV pool supports head_dim from 1 to 256")
        if block_size < 1:
            raise ValueError("block_size must be positive")
        self.n_layer = n_layer
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.n_head = n_head
        self.head_dim = head_dim
        self.groups = -(-head_dim // self.GROUP)
        slab = -(-block_size * self.groups * 34 // 16) * 16
        self.data = torch.empty((n_layer, num_blocks, n_head, slab), dtype=torch.uint8, device=device)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def _parts(self, slabs: torch.Tensor):
        """Views of slabs [..., slab]: K codes and V codes [..., S, g * 16], K scales and V
        scales [..., S, g]."""
        S, g = self.block_size, self.groups
        lead = slabs.shape[:-1]
        codes, scales = S * g * 16, S * g
        k, v = (slabs[..., i * codes:(i + 1) * codes].view(*lead, S, g * 16) for i in range(2))
        ks = slabs[..., 2 * codes:2 * codes + scales].view(*lead, S, g)
        vs = slabs[..., 2 * codes + scales:2 * codes + 2 * scales].view(*lead, g, S).transpose(-1, -2)
        return k, v, ks, vs

    def _encode(self, rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Code bytes [..., g * 16] and scale bytes [..., g] of rows [..., D]."""
        x = torch.nn.functional.pad(rows.float(), (0, self.groups * self.GROUP - self.head_dim))
        x = x.unflatten(-1, (self.groups, self.GROUP))
        top = x.abs().amax(-1)
        lost = ~torch.isfinite(top)
        mantissa, exponent = torch.frexp(torch.where(lost, 1.0, top))
        e = torch.where(top == 0, -125, (exponent - 3 + (mantissa > 0.875).int()).clamp(-125, 125))
        y = torch.ldexp(x.abs(), -e[..., None])
        code = torch.zeros_like(y, dtype=torch.uint8)
        for i, border in enumerate(_E2M1_BORDERS):
            code += y >= border if i % 2 else y > border  # ties to the even code
        code += torch.signbit(x).to(torch.uint8) * 8
        code.masked_fill_(lost[..., None], 0)
        code = code.flatten(-2)
        return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(lost, 255, e + 127).to(torch.uint8)

    def _decode(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        table = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), device=codes.device)
        both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        factor = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
        factor = torch.where(scales == 255, torch.nan, factor)
        x = table[both.int()].unflatten(-1, (self.groups, self.GROUP)) * factor[..., None]
        return x.flatten(-2)[..., :self.head_dim].to(dtype)

    def _put(self, slabs: torch.Tensor, block_offset: int, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        k, v, ks, vs = (p[..., block_offset, :] for p in self._parts(slabs))
        for row, codes, scales in ((k_new, k, ks), (v_new, v, vs)):
            c, s = self._encode(row.to(self.data.device))
            codes.copy_(c)
            scales.copy_(s)

    def write(self, physical_block: int, block_offset: int, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Writes one token slot in every layer; k_new/v_new are [L, H, D]."""
        expected = (self.n_layer, self.n_head, self.head_dim)
        assert tuple(k_new.shape) == expected
        assert tuple(v_new.shape) == expected
        self._put(self.data[:, physical_block], block_offset, k_new, v_new)

    def write_layer(self, layer_idx: int, physical_block: int, block_offset: int, k_new: torch.Tensor,
                    v_new: torch.Tensor) -> None:
        """Writes one token slot of one layer; k_new/v_new are [H, D]."""
        self._put(self.data[layer_idx, physical_block], block_offset, k_new, v_new)

    def gather_sequence(self, seq: SequenceState, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of `seq`'s K/V on the host: two [L, seq.length, H, D] tensors."""
        length, S = seq.length, self.block_size
        n = -(-length // S)
        ids = torch.tensor(list(seq.block_table[:n]), dtype=torch.long, device=self.data.device)
        parts = self._parts(self.data.index_select(1, ids))  # [L, n, H, S, ..]
        out = []
        for codes, scales in (parts[0::2], parts[1::2]):
            x = self._decode(codes, scales, dtype).permute(0, 1, 3, 2, 4).flatten(1, 2)
            out.append(x[:, :length].cpu())
        return out[0], out[1]
