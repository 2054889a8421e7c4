// fp4_kv.hip -- rows of keys and values into the 4-bit pool and back (fp4_kv.h has the
// format and the layout).
//
// Append: with amax = max |x| of a group, the scale is the least 2^e, -125 <= e <= 125,
// with amax <= 7 * 2^e, so that no element is more than half a step from its code (6 stands
// for up to 7), and the code is the nearest value to |x| / 2^e, ties to the even code. From
// amax's bits: e = E - 2 where its mantissa is at most 1.75, else E - 1. All of it is exact
// in f32, so the bits do not depend on how it is computed. A group with an infinity or a
// NaN is NaN (byte 255).
//
// Work split: an "octet" of 8 dims at a time, 4 lanes to a group (their maxima meet by DPP);
// a workgroup takes `rows` whole rows, K and V, a thread kBatch octets at once, whose loads
// are all asked for before anything waits for one. Bound by memory, short calls by the
// chain from a slot to a store. Measured on MI355X (append, gather; us): 8191 rows of 8 heads of 128,
// f16 16.2, 12.0 (42 MB: 2.6, 3.5 TB/s); 256 rows of 32 heads of 128, bf16 5.6, 5.9; 4 of 8 of 32,
// f32 4.4, 3.5.
#include <algorithm>

#include "fp4_kv.h"
#include "minivllm_hip.h"

namespace mgi {
namespace {

constexpr int kRowThreads = 512;
constexpr int kMaxRows = 32;            // rows of a workgroup, at most
constexpr int kBatch = 4;               // octets of a thread in work at once
constexpr int kBitmapWords = 512;       // 16384 bits

// 8 consecutive elements of a row, zeros from dim D on: asked for, then as f32.
template <typename T>
struct Piece {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* row, int64_t sd, int d0, int D, int vec) {
    if (vec) {  // without a branch, whose end would wait for the load
      const uint4* at = reinterpret_cast<const uint4*>(row + (d0 < D ? d0 : 0));
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = at[i];
    } else {
      uint32_t x[2 * sizeof(T)];
#pragma unroll
      for (int i = 0; i < 2 * (int)sizeof(T); ++i) x[i] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (d0 + i < D) {
          const T e = row[(d0 + i) * sd];
          if constexpr (sizeof(T) == 4) x[i] = __float_as_uint(e);
          else x[i / 2] |= (uint32_t)e.bits << (16 * (i & 1));
        }
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
  }
  __device__ __forceinline__ void values(float (&x)[8], bool have) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = have ? __uint_as_float(u[i]) : 0.f;
    } else {
      const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        T e;
        e.bits = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
        x[i] = have ? Elem<T>::load(&e) : 0.f;
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* row, int64_t sd, int d0, int D, int vec, const float (&x)[8]) {
  if (vec) {
    if (d0 >= D) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + d0) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(row + d0 + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        T lo, hi;
        Elem<T>::store(&lo, x[2 * i]);
        Elem<T>::store(&hi, x[2 * i + 1]);
        u[i] = (uint32_t)lo.bits | ((uint32_t)hi.bits << 16);
      }
      *reinterpret_cast<uint4*>(row + d0) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d0 + i < D) Elem<T>::store(row + (d0 + i) * sd, x[i]);
  }
}

// The codes of 8 elements and the group's scale byte; the four lanes of a group call it
// together.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t* byte) {
  uint32_t top = 0;  // max |x| by its bits, which order as the values do; NaN above infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, DPP_QUAD_XOR1, 0xF, 0xF, true));
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, DPP_QUAD_XOR2, 0xF, 0xF, true));
  const bool lost = top >= 0x7f800000u;
  // (top + 0x1fffff) >> 23 is the exponent field, one more where the mantissa passes 1.75.
  const int e = min(max((int)((top + 0x1fffffu) >> 23) - 2, 2), 252);  // of 2^(e - 127)
  *byte = lost ? 255u : (uint32_t)e;
  // The conversion takes each element over 2^(e - 127) to the nearest code, ties to the even
  // one, 6 at most (comparing with the seven borders instead, a long call took 24 us, not 16).
  const float scale = __uint_as_float((uint32_t)e << 23);
  uint32_t codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
  return lost ? 0u : codes;
}

// Where octet `o` of a row is: which of K and V, the head, and its octet in the head's row.
struct Octet {
  int is_v, h, o;
};
__device__ __forceinline__ Octet octet_of(const Fp4RowArgs& a, int u) {
  const int g = u >> 2;                              // group: (K or V, head, group)
  const int kvh = fast_div(g, a.g_mul, a.g_shift, a.groups);
  const int is_v = kvh >= a.H;
  return Octet{is_v, is_v ? kvh - a.H : kvh, ((g - kvh * a.groups) << 2) | (u & 3)};
}

__device__ __forceinline__ int64_t slot_at(const Fp4RowArgs& a, int64_t t) {
  return load_index(a.slots, a.sl_i64, t * a.sl_s);
}

// Where a row's slot is in the pool: its block's bytes and its token there. Found once per row,
// as it takes a 64-bit division.
struct Place {
  int64_t block;
  uint32_t token;
};
__device__ __forceinline__ Place place_of(const Fp4RowArgs& a, int64_t slot) {
  const int64_t blk = slot / a.S;
  return Place{blk * a.p_sn, (uint32_t)(slot - blk * a.S)};
}

// Of rows on one slot the last is kept whole (codes and scale of different rows would be
// neither's values), so each workgroup looks through the slots behind its rows: against a
// bitmap of its own slots first, against the slots themselves where a bit is set.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) fp4_append_kernel(const Fp4RowArgs a) {
  __shared__ int64_t s_slot[kMaxRows];
  __shared__ Place s_place[kMaxRows];
  __shared__ int s_keep[kMaxRows];
  __shared__ uint32_t s_bits[kBitmapWords];
  const int t0 = (int)blockIdx.x * a.rows, rows = min(a.rows, a.T - t0);
  const int tid = (int)threadIdx.x;
  const int octs = 2 * a.H * a.groups * 4, all = rows * octs;  // octets of a row, of all rows
  Piece<T> piece[kBatch];
  // Octets first + i * kRowThreads of the workgroup's; past the last one, the last.
  const auto ask = [&](int first) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = min(first + i * kRowThreads, all - 1), r = fast_div(u, a.o_mul, a.o_shift, octs);
      const Octet at = octet_of(a, u - r * octs);
      const int64_t st = at.is_v ? a.v_st : a.k_st, sh = at.is_v ? a.v_sh : a.k_sh, sd = at.is_v ? a.v_sd : a.k_sd;
      piece[i].load(reinterpret_cast<const T*>(at.is_v ? a.v : a.k) + (t0 + r) * st + at.h * sh, sd, at.o * 8, a.D, a.vec);
    }
  };
  int64_t mine = -1;
  if (tid < rows) mine = slot_at(a, t0 + tid);
  ask(tid);
  for (int i = tid; i < kBitmapWords; i += kRowThreads) s_bits[i] = 0;
  if (tid < rows) {
    if (mine < 0 || mine >= a.N * (int64_t)a.S) mine = -1;
    s_slot[tid] = mine;
    s_place[tid] = place_of(a, mine < 0 ? 0 : mine);
    s_keep[tid] = mine >= 0;
  }
  __syncthreads();
  const auto bit = [](int64_t s) { return ((uint32_t)s * 0x9E3779B1u) >> 18; };
  if (mine >= 0) atomicOr(&s_bits[bit(mine) >> 5], 1u << (bit(mine) & 31));
  __syncthreads();
  for (int first = t0 + 1; first < a.T; first += 4 * kRowThreads) {
    int64_t later[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) later[i] = slot_at(a, min(first + i * kRowThreads + tid, a.T - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = first + i * kRowThreads + tid;
      const uint32_t b = bit(later[i]);
      if (t < a.T && (s_bits[b >> 5] >> (b & 31)) & 1)
        for (int r = 0; r < rows && t0 + r < t; ++r)
          if (s_slot[r] == later[i]) s_keep[r] = 0;
    }
  }
  __syncthreads();
  for (int first = tid; first < all; first += kBatch * kRowThreads) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = min(first + i * kRowThreads, all - 1), r = fast_div(u, a.o_mul, a.o_shift, octs);
      const Octet at = octet_of(a, u - r * octs);
      float x[8];
      piece[i].values(x, at.o * 8 < a.D);
      uint32_t byte;
      const uint32_t codes = encode8(x, &byte);  // by the four lanes of a group together
      if (first + i * kRowThreads >= all || !s_keep[r]) continue;
      const Place to = s_place[r];
      const uint32_t off = to.token, S = a.S, groups = a.groups, g = at.o >> 2;
      unsigned char* slab = a.pool + to.block + at.h * a.p_sh;
      *reinterpret_cast<uint32_t*>(slab + (at.is_v ? fp4_v_codes(S, groups) : 0) + (off * groups * 16 + at.o * 4)) = codes;
      if ((at.o & 3) == 0)
        slab[at.is_v ? fp4_v_scales(S, groups) + g * S + off : fp4_k_scales(S, groups) + off * groups + g] =
            (unsigned char)byte;
    }
    if (first + kBatch * kRowThreads < all) ask(first + kBatch * kRowThreads);
  }
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// Rows of the pool as values; a row whose slot is outside the pool comes out 0.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) fp4_gather_kernel(const Fp4RowArgs a) {
  const int t0 = (int)blockIdx.x * a.rows, rows = min(a.rows, a.T - t0);
  const int octs = 2 * a.H * a.groups * 4, all = rows * octs;
  const uint32_t S = a.S, groups = a.groups;
  __shared__ Place s_place[kMaxRows];
  __shared__ int s_inside[kMaxRows];
  if ((int)threadIdx.x < rows) {
    const int64_t slot = slot_at(a, t0 + (int)threadIdx.x);
    const bool inside = slot >= 0 && slot < a.N * (int64_t)a.S;
    s_place[threadIdx.x] = place_of(a, inside ? slot : 0);
    s_inside[threadIdx.x] = inside;
  }
  __syncthreads();
  for (int first = (int)threadIdx.x; first < all; first += kBatch * kRowThreads) {
    uint32_t codes[kBatch], byte[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = min(first + i * kRowThreads, all - 1), r = fast_div(u, a.o_mul, a.o_shift, octs);
      const Octet at = octet_of(a, u - r * octs);
      const Place from = s_place[r];
      const uint32_t off = from.token, g = at.o >> 2;
      const unsigned char* slab = a.pool + from.block + at.h * a.p_sh;
      codes[i] = *reinterpret_cast<const uint32_t*>(slab + (at.is_v ? fp4_v_codes(S, groups) : 0) + (off * groups * 16 + at.o * 4));
      byte[i] = slab[at.is_v ? fp4_v_scales(S, groups) + g * S + off : fp4_k_scales(S, groups) + off * groups + g];
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = first + i * kRowThreads, r = fast_div(min(u, all - 1), a.o_mul, a.o_shift, octs);
      const Octet at = octet_of(a, min(u, all - 1) - r * octs);
      const float scale = __uint_as_float(byte[i] << 23);  // 255: the conversion gives NaN
      const f32x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 0);
      const f32x2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 1);
      const f32x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 2);
      const f32x2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 3);
      float x[8] = {p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
      if (!s_inside[r]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
      }
      const int64_t st = at.is_v ? a.v_st : a.k_st, sh = at.is_v ? a.v_sh : a.k_sh, sd = at.is_v ? a.v_sd : a.k_sd;
      if (u < all)
        store8(reinterpret_cast<T*>(at.is_v ? a.v : a.k) + (t0 + r) * st + at.h * sh, sd, at.o * 8, a.D, a.vec, x);
    }
  }
}

// Rows per workgroup: one octet for each thread at least; more than 512 workgroups take
// more rows each, up to kMaxRows.
int rows_per_workgroup(const Fp4RowArgs& a) {
  const int octs = 2 * a.H * a.groups * 4, least = (kRowThreads + octs - 1) / octs, rows = (a.T + 511) / 512;
  return std::min(std::max(rows, least), kMaxRows);
}

template <typename F>
hipError_t launch_rows(F* kernel, Fp4RowArgs a, hipStream_t stream) {
  if (a.T <= 0) return hipSuccess;
  a.rows = rows_per_workgroup(a);
  void* args[] = {&a};
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((unsigned)((a.T + a.rows - 1) / a.rows)),
                         dim3(kRowThreads), args, 0, stream);
}

}  // namespace

// Rows of a launch: what looking through the later rows' slots costs grows with their square, and
// of two launches the later one's rows are kept by itself. 131072 rows of 8 heads of 128, bf16, slots in
// random order: 493 us in one launch, 316 by 32768 rows, 372 by 16384 (32768 rows: 68, and 81).
constexpr int kAppendRows = 32768;

hipError_t launch_fp4_append(const Fp4RowArgs& a, int dtype, hipStream_t stream) {
  for (int t = 0; t < a.T; t += kAppendRows) {
    const int64_t bytes = dtype == MGI_F32 ? 4 : 2;
    Fp4RowArgs part = a;
    part.T = std::min(a.T - t, kAppendRows);
    part.k = static_cast<char*>(a.k) + t * a.k_st * bytes;
    part.v = static_cast<char*>(a.v) + t * a.v_st * bytes;
    part.slots = static_cast<const char*>(a.slots) + t * a.sl_s * (a.sl_i64 ? 8 : 4);
    const hipError_t e = dtype == MGI_F32    ? launch_rows(&fp4_append_kernel<float>, part, stream)
                         : dtype == MGI_BF16 ? launch_rows(&fp4_append_kernel<bf16_t>, part, stream)
                                             : launch_rows(&fp4_append_kernel<f16_t>, part, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_fp4_gather(const Fp4RowArgs& a, int dtype, hipStream_t stream) {
  return dtype == MGI_F32    ? launch_rows(&fp4_gather_kernel<float>, a, stream)
         : dtype == MGI_BF16 ? launch_rows(&fp4_gather_kernel<bf16_t>, a, stream)
                             : launch_rows(&fp4_gather_kernel<f16_t>, a, stream);
}

}  // namespace mgi
