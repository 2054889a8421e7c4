// fp4_kv.h -- the 4-bit KV pool: where a token's codes and scales are, and the
// arguments of the kernels that write, read and attend over it (fp4_kv.hip,
// paged_fp4.h).
//
// A head's row of D dims is cut into groups of 32 (the last padded with zeros): 4-bit
// e2m1 codes (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and
// one e8m0 byte for the group (2^(byte - 127); 255: the whole group is NaN), which are the
// OCP microscaling formats gfx950 converts in hardware. One (layer, block, head) is one
// slab of bytes, so a wavefront that attends over a block reads one contiguous piece:
//   K codes  [S][groups * 16]   two codes to a byte, the even dim in the low half
//   V codes  [S][groups * 16]
//   K scales [S][groups]        a lane's key group is one byte beside its neighbours'
//   V scales [groups][S]        the scales of four consecutive tokens are one word
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "mgi_common.h"

namespace mgi {

constexpr int kFp4Group = 32;
constexpr int kFp4MaxDim = 256;
constexpr float kFp4Slack = 8.f;  // log2: a score may pass the running maximum by this before it moves

__host__ __device__ inline int64_t fp4_groups(int64_t D) { return (D + kFp4Group - 1) / kFp4Group; }
// Bytes of one (layer, block, head), a multiple of 16.
__host__ __device__ inline int64_t fp4_slab_bytes(int64_t S, int64_t D) {
  return (S * fp4_groups(D) * 34 + 15) / 16 * 16;
}
__host__ __device__ inline uint32_t fp4_v_codes(uint32_t S, uint32_t groups) { return S * groups * 16; }
__host__ __device__ inline uint32_t fp4_k_scales(uint32_t S, uint32_t groups) { return S * groups * 32; }
__host__ __device__ inline uint32_t fp4_v_scales(uint32_t S, uint32_t groups) { return S * groups * 33; }

// Rows into the pool (append), or out of it (gather). Strides of k and v in elements,
// of the pool in bytes; the pool pointer already points at the layer.
struct Fp4RowArgs {
  unsigned char* pool;
  int64_t p_sn, p_sh;
  void* k;
  void* v;
  int64_t k_st, k_sh, k_sd;
  int64_t v_st, v_sh, v_sd;
  const void* slots;
  int64_t sl_s;
  int sl_i64;
  int T, H, D, S, groups;
  int64_t N;
  int vec;              // rows contiguous and 16-byte aligned, D a multiple of 8
  int rows;             // rows per workgroup
  uint32_t g_mul, o_mul;  // divisions by groups and by the row's octets (magic_of)
  int g_shift, o_shift;
};
hipError_t launch_fp4_append(const Fp4RowArgs& a, int dtype, hipStream_t stream);
hipError_t launch_fp4_gather(const Fp4RowArgs& a, int dtype, hipStream_t stream);

// bf16 terms of a query element: 1 for bf16, 2 for f16, 3 for f32.
__host__ __device__ constexpr int fp4_query_terms(int bytes, bool is_bf16) { return bytes == 4 ? 3 : is_bf16 ? 1 : 2; }
// Wavefronts per SIMD that the decode kernels' registers allow without spilling a vector
// register: 4 registers per group for each query term and each of two accumulators, and the tile's own.
// More wavefronts hide more of the loads: 64 x 512-4096 tokens, 32 heads of 128, bf16 took 150 us at
// two, 131 at three.
__host__ __device__ constexpr int fp4_occupancy(int groups, int query_terms) {
  return groups * (2 + query_terms) <= 8    ? 4
         : groups * (2 + query_terms) <= 12 ? 3
         : groups * (2 + query_terms) <= 32 ? 2
                                            : 1;
}
// Wavefronts of a workgroup of the one-launch form, at most.
__host__ __device__ constexpr int fp4_one_waves(int groups, int query_terms) {
  return fp4_occupancy(groups, query_terms) > 1 ? 8 : 4;
}

// Decode attention over the pool (paged_fp4.h).
struct Fp4DecodeArgs {
  void* out;
  int64_t o_sb, o_sh, o_sd;
  const void* q;
  int64_t q_sb, q_sh, q_sd;
  const unsigned char* pool;
  int64_t p_sn, p_sh;
  const void* bt;
  int64_t bt_sb, bt_sm;
  const void* cl;
  int64_t cl_s;
  int bt_i64, cl_i64;
  int B, Hk, G, D, S, M;   // G query heads per KV head
  int64_t N;
  int q_tiles;             // tiles of 16 query heads per KV head
  float scale_log2;        // |scale| * log2(e) (1 for a scale of 0)
  float slack;             // the running maximum moves when a score, before the scale, passes it by this
  uint32_t q_flip;         // sign bit of q, for a negative scale
  int q_zero;              // scale is 0
  int vec;                 // q and out rows contiguous and 16-byte aligned, D a multiple of 8
  uint32_t s_mul;          // division by S (magic_of)
  int s_shift;
  int one_launch;          // a workgroup of `waves` wavefronts per (sequence, KV head)
  int waves;               // otherwise: wavefronts of the whole launch, a multiple of 4
  float* ws_acc;           // [2 * waves][min(G, 16)][groups * 32]
  float2* ws_ml;           // [2 * waves][16]  (max, before the scale, and sum)
  int* ws_cum;             // [B + 1] exclusive prefix sums of tiles per sequence
};
hipError_t launch_paged_fp4_f32(const Fp4DecodeArgs& a, hipStream_t stream);
hipError_t launch_paged_fp4_bf16(const Fp4DecodeArgs& a, hipStream_t stream);
hipError_t launch_paged_fp4_f16(const Fp4DecodeArgs& a, hipStream_t stream);

}  // namespace mgi
