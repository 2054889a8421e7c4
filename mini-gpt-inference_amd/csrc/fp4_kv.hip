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
// Work split: an "octet" of 8 dims per thread, 4 lanes to a group (their maxima meet by
// DPP); a workgroup takes `rows` whole rows, K and V.
#include "fp4_kv.h"
#include "minivllm_hip.h"

namespace mgi {
namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxRows = 32;            // rows of a workgroup, at most
constexpr int kBitmapWords = 512;       // 16384 bits

// 8 consecutive elements of a row as f32, zeros from dim D on.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t sd, int d0, int D, int vec, float (&x)[8]) {
  if (vec) {
    if (d0 >= D) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    } else if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + d0), b = *reinterpret_cast<const float4*>(row + d0 + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(row + d0);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        T e;
        e.bits = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
        x[i] = Elem<T>::load(&e);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = d0 + i < D ? Elem<T>::load(row + (d0 + i) * sd) : 0.f;
  }
}

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

// The code of |x| / 2^e for y = |x| / 2^e: how many of the borders between neighbouring
// values lie below it. A border itself goes to the even code.
__device__ __forceinline__ uint32_t e2m1_code(float y) {
  return (uint32_t)(y > 0.25f) + (y >= 0.75f) + (y > 1.25f) + (y >= 1.75f) + (y > 2.5f) + (y >= 3.5f) + (y > 5.f);
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
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e), exact
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    codes |= (e2m1_code(fabsf(x[i]) * inv) | (__float_as_uint(x[i]) >> 31 << 3)) << (4 * i);
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

// Of rows on one slot the last is kept whole (codes and scale of different rows would be
// neither's values), so each workgroup looks through the slots behind its rows: against a
// bitmap of its own slots first, against the slots themselves where a bit is set.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) fp4_append_kernel(const Fp4RowArgs a) {
  __shared__ int64_t s_slot[kMaxRows];
  __shared__ int s_keep[kMaxRows];
  __shared__ uint32_t s_bits[kBitmapWords];
  const int t0 = (int)blockIdx.x * a.rows, rows = min(a.rows, a.T - t0);
  const int tid = (int)threadIdx.x;
  for (int i = tid; i < kBitmapWords; i += kRowThreads) s_bits[i] = 0;
  int64_t mine = -1;
  if (tid < rows) {
    mine = slot_at(a, t0 + tid);
    if (mine < 0 || mine >= a.N * (int64_t)a.S) mine = -1;
    s_slot[tid] = mine;
    s_keep[tid] = mine >= 0;
  }
  __syncthreads();
  const auto bit = [](int64_t s) { return ((uint32_t)s * 0x9E3779B1u) >> 18; };
  if (mine >= 0) atomicOr(&s_bits[bit(mine) >> 5], 1u << (bit(mine) & 31));
  __syncthreads();
  for (int t = t0 + 1 + tid; t < a.T; t += kRowThreads) {
    const int64_t s = slot_at(a, t);
    const uint32_t b = bit(s);
    if ((s_bits[b >> 5] >> (b & 31)) & 1)
      for (int r = 0; r < rows && t0 + r < t; ++r)
        if (s_slot[r] == s) s_keep[r] = 0;
  }
  __syncthreads();
  const int octs = 2 * a.H * a.groups * 4;  // octets of a row
  for (int u = tid; u < rows * octs; u += kRowThreads) {
    const int r = fast_div(u, a.o_mul, a.o_shift, octs);
    const Octet at = octet_of(a, u - r * octs);
    if (!s_keep[r]) continue;  // the same for the four lanes of a group
    const int64_t st = at.is_v ? a.v_st : a.k_st, sh = at.is_v ? a.v_sh : a.k_sh, sd = at.is_v ? a.v_sd : a.k_sd;
    const T* row = reinterpret_cast<const T*>(at.is_v ? a.v : a.k) + (t0 + r) * st + at.h * sh;
    float x[8];
    load8(row, sd, at.o * 8, a.D, a.vec, x);
    uint32_t byte;
    const uint32_t codes = encode8(x, &byte);
    const int64_t s = s_slot[r], blk = s / a.S;
    const uint32_t off = (uint32_t)(s - blk * a.S), S = a.S, groups = a.groups, g = at.o >> 2;
    unsigned char* slab = a.pool + blk * a.p_sn + at.h * a.p_sh;
    *reinterpret_cast<uint32_t*>(slab + (at.is_v ? fp4_v_codes(S, groups) : 0) + (off * groups * 16 + at.o * 4)) = codes;
    if ((at.o & 3) == 0)
      slab[at.is_v ? fp4_v_scales(S, groups) + g * S + off : fp4_k_scales(S, groups) + off * groups + g] =
          (unsigned char)byte;
  }
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// Rows of the pool as values; a row whose slot is outside the pool comes out 0.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) fp4_gather_kernel(const Fp4RowArgs a) {
  const int t0 = (int)blockIdx.x * a.rows, rows = min(a.rows, a.T - t0);
  const int octs = 2 * a.H * a.groups * 4;
  for (int u = (int)threadIdx.x; u < rows * octs; u += kRowThreads) {
    const int r = fast_div(u, a.o_mul, a.o_shift, octs);
    const Octet at = octet_of(a, u - r * octs);
    const int64_t s = slot_at(a, t0 + r);
    const bool inside = s >= 0 && s < a.N * (int64_t)a.S;
    const int64_t blk = inside ? s / a.S : 0;
    const uint32_t off = inside ? (uint32_t)(s - blk * a.S) : 0u, S = a.S, groups = a.groups, g = at.o >> 2;
    const unsigned char* slab = a.pool + blk * a.p_sn + at.h * a.p_sh;
    const uint32_t codes =
        *reinterpret_cast<const uint32_t*>(slab + (at.is_v ? fp4_v_codes(S, groups) : 0) + (off * groups * 16 + at.o * 4));
    const uint32_t byte =
        slab[at.is_v ? fp4_v_scales(S, groups) + g * S + off : fp4_k_scales(S, groups) + off * groups + g];
    const float scale = __uint_as_float(byte << 23);  // 255: the conversion gives NaN
    float x[8];
    const f32x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
    const f32x2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
    const f32x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
    const f32x2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
    x[0] = p0[0], x[1] = p0[1], x[2] = p1[0], x[3] = p1[1], x[4] = p2[0], x[5] = p2[1], x[6] = p3[0], x[7] = p3[1];
    if (!inside) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
    const int64_t st = at.is_v ? a.v_st : a.k_st, sh = at.is_v ? a.v_sh : a.k_sh, sd = at.is_v ? a.v_sd : a.k_sd;
    store8(reinterpret_cast<T*>(at.is_v ? a.v : a.k) + (t0 + r) * st + at.h * sh, sd, at.o * 8, a.D, a.vec, x);
  }
}

// Rows per workgroup: about 1024 octets, four to a thread; more where that leaves more
// than 4 workgroups per CU, up to kMaxRows.
int rows_per_workgroup(const Fp4RowArgs& a) {
  const int octs = 2 * a.H * a.groups * 4;
  int rows = octs >= 1024 ? 1 : 1024 / octs;
  while (rows < kMaxRows && (a.T + rows - 1) / rows > 1024) ++rows;
  return rows < kMaxRows ? rows : kMaxRows;
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

hipError_t launch_fp4_append(const Fp4RowArgs& a, int dtype, hipStream_t stream) {
  return dtype == MGI_F32    ? launch_rows(&fp4_append_kernel<float>, a, stream)
         : dtype == MGI_BF16 ? launch_rows(&fp4_append_kernel<bf16_t>, a, stream)
                             : launch_rows(&fp4_append_kernel<f16_t>, a, stream);
}

hipError_t launch_fp4_gather(const Fp4RowArgs& a, int dtype, hipStream_t stream) {
  return dtype == MGI_F32    ? launch_rows(&fp4_gather_kernel<float>, a, stream)
         : dtype == MGI_BF16 ? launch_rows(&fp4_gather_kernel<bf16_t>, a, stream)
                             : launch_rows(&fp4_gather_kernel<f16_t>, a, stream);
}

}  // namespace mgi
