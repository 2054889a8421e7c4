// rope.hip -- RMS norms of query and key heads with the position rotation, and
// the KV append that rotates on the way, for gfx950.
//
// A head row x of D elements becomes
//   y = x * rsqrt(mean_d x_d^2 + eps) * w           (with weights; else y = x)
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)    for the R/2 pairs (i, j)
// with c, s = cos, sin of pair p's angle, cos_sin[position, p] and
// cos_sin[position, R/2 + p]; pair p is (p, p + R/2), or (2p, 2p + 1)
// interleaved. Dims R .. D-1 are not rotated. All of it in f32, rounded once to
// the type stored: a head row is read once and stays in registers.
//
// Bound by memory on long calls and by one launch on short ones, so nothing is
// staged: a lane holds two chunks of a head row that a rotation needs together
// (dims C p .. C p + C-1 and the same plus R/2), loads them with one instruction
// each and shares only the sum of squares, over the lanes of the head. Everything
// but the angles loads at once, the angles once the position is there, and no load is
// under a condition: its end would wait for all of them. 8192 rows of 32 + 8 bf16 heads
// of 128 take 28 us on cached inputs (6.1 TB/s) and 33 from memory (5.2; a large copy
// 4.9). With conditions, 64-bit offsets and rounding by hand: 37 and 43; in that form
// two head rows to a lane took 2 % more, four 29 % (more registers, fewer wavefronts),
// and a workgroup per row walking its heads 75 %. 13 rows appended take 3.1 us (5.6-6.2
// with the host's call), 256 rows of 32 + 2 x 32 heads 5.0; without a look at the later
// rows' slots (LaterRows) 2.8 and 4.5.
#include <type_traits>

#include "mgi_common.h"
#include "mgi_internal.h"
#include "minivllm_hip.h"

namespace mgi {

constexpr int kRopeThreads = 256;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// N consecutive elements from f32, with one rounding each. Pointers are aligned to the
// chunk's bytes, 16 at most.
template <int N>
__device__ __forceinline__ void store_chunk(float* p, const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
template <int N, typename T>
__device__ __forceinline__ void store_chunk(T* p, const float (&x)[N]) {
  using Two = std::conditional_t<std::is_same_v<T, bf16_t>, bf16x2, f16x2>;
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, Two));
  if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
// Where row t's key and value go: the pool's slot, or row t of k_out (no v).
// False when nothing is to be written.
__device__ __forceinline__ bool rope_target(const RopeArgs& a, int64_t t, bool placed, int64_t* k_off, int64_t* v_off) {
  if (!a.slots) {
    *k_off = t * a.ko_st;
    return true;
  }
  const int64_t slot = load_index(a.slots, a.sl_i64, t * a.sl_s);
  if (!placed || slot < 0 || slot >= a.N * (int64_t)a.S) return false;
  const int64_t blk = slot / a.S, off = slot - blk * a.S;
  *k_off = blk * a.ko_sn + off * a.ko_st;
  *v_off = blk * a.vo_sn + off * a.vo_st;
  return true;
}

__device__ __forceinline__ float weight_at(const void* w, int f32, int dtype, int64_t i) {
  if (f32) return ((const float*)w)[i];
  return dtype == MGI_BF16 ? bf16_to_f32(((const uint16_t*)w)[i]) : f16_to_f32(((const uint16_t*)w)[i]);
}

// A chunk as loaded, and as f32.
template <typename T, int C>
struct Raw {
  uint32_t w[C * (int)sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(w) == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(w) == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else if constexpr (std::is_same_v<T, bf16_t>) return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
    else return f16_to_f32((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
  }
};

// A value converted as the append without rotation converts it, NaN included.
template <int N, typename T>
__device__ __forceinline__ void store_value(T* p, const float (&x)[N]) {
  if constexpr (std::is_same_v<T, bf16_t>) {
    Raw<bf16_t, N> r;
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      r.w[i] = (uint32_t)f32_to_bf16(x[2 * i]) | ((uint32_t)f32_to_bf16(x[2 * i + 1]) << 16);
    r.store(p);
  } else {
    store_chunk(p, x);
  }
}

// The sum over aligned groups of gp lanes, gp a power of two.
__device__ __forceinline__ float group_sum(float x, int gp) {
  if (gp > 1) x += dpp<DPP_QUAD_XOR1>(x);
  if (gp > 2) x += dpp<DPP_QUAD_XOR2>(x);
  if (gp > 4) x += dpp<DPP_ROW_HALF_MIRROR>(x);
  if (gp > 8) x += dpp<DPP_ROW_MIRROR>(x);
  if (gp > 16) x += swizzle_xor16(x);
  if (gp > 32) x += __shfl_xor(x, 32, 64);
  return x;
}

// Rows on one slot: a slot's head rows are many wavefronts', K and V apart, and nothing
// orders two rows' stores, so left alone a slot may hold heads (or 16-byte pieces) of
// one row and of the other. In calls of up to kOrderedRows rows every wavefront looks
// through the later rows' slots and leaves out a row that one of them replaces: K and V
// are the last row's, whole. 256 slots are 2 KB, no more than a wavefront's own eight head
// rows of 128, and load beside them; a long chunk's would be many times that, so longer
// calls do not look.
constexpr int kOrderedRows = 256;

// The low words of the slots of a wavefront's rows (t is its first lane's, the lowest)
// and of those after them: lane l holds rows l, l + 64, ...
struct LaterRows {
  uint32_t low[kOrderedRows / 64];
  __device__ __forceinline__ static bool holds(const RopeArgs& a, int i, int t) { return 64 * i < a.T && 64 * i + 63 > t; }
  __device__ __forceinline__ void load(const RopeArgs& a, int t) {
    const int first = __builtin_amdgcn_readfirstlane(t), lane = (int)threadIdx.x & 63;
    const char* p = (const char*)a.slots;
#pragma unroll
    for (int i = 0; i < kOrderedRows / 64; ++i)
      if (holds(a, i, first))
        low[i] = *(const uint32_t*)(p + (((uint64_t)min(lane + 64 * i, a.T - 1) * (uint64_t)a.sl_s) << (a.sl_i64 ? 3 : 2)));
  }
  // For the lanes that ask: whether a row after theirs is written to their slot. Every
  // lane of the wavefront takes part.
  __device__ __forceinline__ bool replace(const RopeArgs& a, int t, int64_t slot, bool asks) const {
    const int first = __builtin_amdgcn_readfirstlane(t), lane = (int)threadIdx.x & 63;
    bool out = false;
    for (uint64_t left = __ballot(asks); left;) {  // a row at a time
      const int src = __builtin_ctzll(left), row = __builtin_amdgcn_readlane(t, src);
      const uint32_t want = (uint32_t)__builtin_amdgcn_readlane((int)slot, src);
      uint32_t same = 0;
#pragma unroll
      for (int i = 0; i < kOrderedRows / 64; ++i)
        if (holds(a, i, first)) same |= (low[i] == want && lane + 64 * i > row && lane + 64 * i < a.T ? 1u : 0u) << i;
      bool hit = false;
      for (; same; same &= same - 1) {  // the rest of the slot, and its row's position
        const int64_t r = lane + 64 * __builtin_ctz(same);
        const int64_t pos = load_index(a.positions, a.pos_i64, r * a.pos_s);
        const uint32_t high = (uint32_t)__builtin_amdgcn_readlane((int)(slot >> 32), src);
        hit |= (uint32_t)(load_index(a.slots, a.sl_i64, r * a.sl_s) >> 32) == high &&
               pos >= 0 && pos < a.P;  // without angles a row is not written
      }
      const bool hits = __any(hit);
      if (t == row) out = hits;
      left &= ~__ballot(t == row);
    }
    return out;
  }
};

// n * stride, both below 2^31: one instruction, where a 64-bit stride takes three of a
// quarter of the rate.
__device__ __forceinline__ uint64_t times(int n, int64_t stride) { return (uint64_t)(uint32_t)n * (uint32_t)stride; }

// TI: q, k, v; TO: q_out and the keys' and values' target. C: elements per chunk. All
// strides, positions and slots are below 2^31. ORDERED: of rows on one slot the last.
template <typename TI, typename TO, int C, bool INTER, bool ORDERED>
__global__ void __launch_bounds__(kRopeThreads) rope_vec(const RopeArgs a) {
  const int gp = 1 << a.gp_shift;  // lanes per head row
  const int sub = (int)threadIdx.x & (gp - 1), slots = (int)blockDim.x >> a.gp_shift;
  const int heads = a.Hq + a.Hk + a.Hv, total = a.T * heads;
  // The lane's two chunks: R / 2 apart inside the rotated dims, half of the
  // others apart past them. Lanes and items too many load item 0's first dims.
  const int half = a.R >> 1, rot = half / C, rest = (a.D - a.R) >> 1;
  const int item = (int)blockIdx.x * slots + ((int)threadIdx.x >> a.gp_shift);
  const bool in = item < total, mine = in && sub < a.D / (2 * C), turns = sub < rot;
  const int d0 = turns ? sub * C : mine ? a.R + (sub - rot) * C : 0, d1 = d0 + (turns ? half : mine ? rest : 0);
  const int t = in ? fast_div(item, a.h_mul, a.h_shift, heads) : 0, h = in ? item - t * heads : 0;
  const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
  const int hh = is_q ? h : is_v ? h - a.Hq - a.Hk : h - a.Hq;
  // These loads are under no condition, so that waiting for the position leaves the
  // others on their way.
  Index at_pos, at_slot;
  at_pos.load(a.positions, a.pos_i64, times(t, a.pos_s));
  at_slot.load(a.slots ? a.slots : a.positions, a.slots ? a.sl_i64 : a.pos_i64, times(t, a.slots ? a.sl_s : a.pos_s));
  Raw<TI, C> x[2];
  const TI* src = (const TI*)(is_q ? a.q : is_v ? a.v : a.k);
  src += times(t, is_q ? a.q_st : is_v ? a.v_st : a.k_st) + times(hh, is_q ? a.q_sh : is_v ? a.v_sh : a.k_sh);
  x[0].load(src + d0);
  x[1].load(src + d1);
  LaterRows later;
  if constexpr (ORDERED) later.load(a, t);
  const int64_t pos = at_pos.value(a.pos_i64), slot = at_slot.value(a.sl_i64);
  const bool placed = pos >= 0 && pos < a.P;
  // Half-split: pairs (d0 + i, d1 + i) with cs[i]. Interleaved: pair i of the
  // first chunk with cs[i], of the second with cs[C/2 + i].
  float cs[C], sn[C];
  const float* line = a.table + times(placed ? (int)pos : 0, a.table_s);
  const int a0 = turns ? d0 : 0, a1 = turns ? d1 : half;  // lanes without pairs load some angles
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int p = INTER ? (i < C / 2 ? a0 / 2 + i : a1 / 2 + i - C / 2) : a0 + i;
    cs[i] = line[p], sn[i] = line[half + p];
  }
  // The norm's weights as loaded: C words of f32, else C / 2.
  uint32_t wr[2][C];
  if (a.qw) {
    const void* p = is_q ? a.qw : a.kw;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int d = s ? d1 : d0;
      if (a.w_f32) {
#pragma unroll
        for (int i = 0; i < C; i += 4) {
          const uint4 v = *(const uint4*)((const float*)p + d + i);
          wr[s][i] = v.x, wr[s][i + 1] = v.y, wr[s][i + 2] = v.z, wr[s][i + 3] = v.w;
        }
      } else if constexpr (sizeof(TI) == 2) {
        Raw<TI, C> r;
        r.load((const TI*)p + d);
#pragma unroll
        for (int i = 0; i < C / 2; ++i) wr[s][i] = r.w[i];
      }
    }
  }
  // Where the row goes: q_out, or k_out or the pools.
  TO* dst = (TO*)(is_q ? a.q_out : is_v ? a.v_out : a.k_out);
  bool keeps = mine, replaced = false;
  if constexpr (ORDERED) replaced = later.replace(a, t, slot, mine && !is_q);
  if (is_q || !a.slots) {
    dst += times(t, is_q ? a.qo_st : a.ko_st) + times(hh, is_q ? a.qo_sh : a.ko_sh);
  } else {
    keeps = mine && placed && !replaced && slot >= 0 && slot < a.N * (int64_t)a.S;
    const int at = keeps ? (int)slot : 0, blk = fast_div(at, a.s_mul, a.s_shift, a.S);
    dst += times(blk, is_v ? a.vo_sn : a.ko_sn) + times(at - blk * a.S, is_v ? a.vo_st : a.ko_st) +
           times(hh, is_v ? a.vo_sh : a.ko_sh);
  }
  if (is_v) {
    if (!keeps) return;
    if constexpr (std::is_same_v<TI, TO>) {  // a copy, bit for bit
      x[0].store(dst + d0);
      x[1].store(dst + d1);
    } else {
      float y[2][C];
#pragma unroll
      for (int i = 0; i < C; ++i) y[0][i] = x[0][i], y[1][i] = x[1][i];
      store_value(dst + d0, y[0]);
      store_value(dst + d1, y[1]);
    }
    return;
  }
  float z[2][C];
#pragma unroll
  for (int i = 0; i < C; ++i) z[0][i] = x[0][i], z[1][i] = x[1][i];
  float r = 1.f;
  if (a.qw) {  // lanes without chunks only pass the others' sums on
    float ss = 0.f;
    if (mine) {
#pragma unroll
      for (int i = 0; i < C; ++i) ss = fmaf(z[0][i], z[0][i], fmaf(z[1][i], z[1][i], ss));
    }
    ss = group_sum(ss, gp);
    r = rsqrtf(ss * a.inv_d + a.eps);
  }
  if (!keeps) return;
  if (turns && !placed) r = __builtin_nanf("");  // a query without angles
  if (a.qw) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float w[C];
#pragma unroll
      for (int i = 0; i < C; ++i) w[i] = __uint_as_float(wr[s][i]);
      if constexpr (sizeof(TI) == 2) {
        if (!a.w_f32) {
          Raw<TI, C> raw;
#pragma unroll
          for (int i = 0; i < C / 2; ++i) raw.w[i] = wr[s][i];
#pragma unroll
          for (int i = 0; i < C; ++i) w[i] = raw[i];
        }
      }
#pragma unroll
      for (int i = 0; i < C; ++i) z[s][i] = z[s][i] * r * w[i];
    }
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < C; ++i) z[s][i] *= r;
  }
  if (turns) {  // past the rotated dims: as it is (an infinity times 0 is no 0)
    if constexpr (INTER) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
          const float c = cs[s * C / 2 + i], n = sn[s * C / 2 + i], p = z[s][2 * i], q = z[s][2 * i + 1];
          z[s][2 * i] = p * c - q * n;
          z[s][2 * i + 1] = q * c + p * n;
        }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float p = z[0][i], q = z[1][i];
        z[0][i] = p * cs[i] - q * sn[i];
        z[1][i] = q * cs[i] + p * sn[i];
      }
    }
  }
  store_chunk(dst + d0, z[0]);
  store_chunk(dst + d1, z[1]);
}

// Any strides and any even R: one wavefront per head row, lanes over the dims.
template <typename TI, typename TO, bool ORDERED>
__global__ void __launch_bounds__(kRopeThreads) rope_any(const RopeArgs a) {
  const int heads = a.Hq + a.Hk + a.Hv;
  const int64_t unit = (int64_t)blockIdx.x * (kRopeThreads / 64) + threadIdx.x / 64;
  if (unit >= (int64_t)a.T * heads) return;
  const int64_t t = unit / heads;
  const int h = (int)(unit - t * heads), lane = (int)threadIdx.x & 63;
  const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
  const int hh = is_q ? h : is_v ? h - a.Hq - a.Hk : h - a.Hq;
  const int64_t pos = load_index(a.positions, a.pos_i64, t * a.pos_s);
  const bool placed = pos >= 0 && pos < a.P;
  int64_t k_off = 0, v_off = 0;
  if (!rope_target(a, t, placed, &k_off, &v_off) && !is_q) return;
  if constexpr (ORDERED) {
    if (!is_q) {
      LaterRows later;
      later.load(a, (int)t);
      if (later.replace(a, (int)t, load_index(a.slots, a.sl_i64, t * a.sl_s), true)) return;
    }
  }
  const TI* src = is_q   ? (const TI*)a.q + t * a.q_st + (int64_t)hh * a.q_sh
                  : is_v ? (const TI*)a.v + t * a.v_st + (int64_t)hh * a.v_sh
                         : (const TI*)a.k + t * a.k_st + (int64_t)hh * a.k_sh;
  const int64_t ss = is_q ? a.q_sd : is_v ? a.v_sd : a.k_sd;
  TO* dst = is_q   ? (TO*)a.q_out + t * a.qo_st + (int64_t)hh * a.qo_sh
            : is_v ? (TO*)a.v_out + v_off + (int64_t)hh * a.vo_sh
                   : (TO*)a.k_out + k_off + (int64_t)hh * a.ko_sh;
  const int64_t ds = is_q ? a.qo_sd : is_v ? a.vo_sd : a.ko_sd;
  if (is_v) {
    for (int d = lane; d < a.D; d += 64) {
      if constexpr (std::is_same_v<TI, TO>) dst[d * ds] = src[d * ss];
      else Elem<TO>::store(dst + d * ds, Elem<TI>::load(src + d * ss));
    }
    return;
  }
  float r = 1.f;
  const void* w = is_q ? a.qw : a.kw;
  if (w) {
    float sum = 0.f;
    for (int d = lane; d < a.D; d += 64) {
      const float x = Elem<TI>::load(src + d * ss);
      sum = fmaf(x, x, sum);
    }
    r = 1.0f / sqrtf(wave_sum(sum) * a.inv_d + a.eps);
  }
  auto normed = [&](int d) {
    const float x = Elem<TI>::load(src + d * ss);
    return w ? x * r * weight_at(w, a.w_f32, a.dtype, d) : x;
  };
  const int half = a.R >> 1;
  for (int d = lane; d < a.D; d += 64) {
    float y = normed(d);
    if (d < a.R) {
      const int p = a.interleaved ? d >> 1 : d < half ? d : d - half;
      const bool first = a.interleaved ? !(d & 1) : d < half;
      const float other = normed(a.interleaved ? d ^ 1 : first ? d + half : d - half);
      const float* row = a.table + (placed ? pos : 0) * a.table_s;
      const float c = placed ? row[p] : __builtin_nanf(""), s = placed ? row[half + p] : __builtin_nanf("");
      y = first ? y * c - other * s : y * c + other * s;
    }
    Elem<TO>::store(dst + d * ds, y);
  }
}

namespace {

template <typename TI, typename TO, bool ORDERED>
const void* rope_kernel(int chunk, int interleaved) {
  if (chunk == 0) return (const void*)&rope_any<TI, TO, ORDERED>;
  if constexpr (sizeof(TI) == 2)
    if (chunk == 8)
      return interleaved ? (const void*)&rope_vec<TI, TO, 8, true, ORDERED>
                         : (const void*)&rope_vec<TI, TO, 8, false, ORDERED>;
  return interleaved ? (const void*)&rope_vec<TI, TO, 4, true, ORDERED>
                     : (const void*)&rope_vec<TI, TO, 4, false, ORDERED>;
}
template <typename TI, typename TO>
const void* rope_kernel(const RopeArgs& a) {
  return a.slots && a.T > 1 && a.T <= kOrderedRows ? rope_kernel<TI, TO, true>(a.chunk, a.interleaved)
                                                   : rope_kernel<TI, TO, false>(a.chunk, a.interleaved);
}

}  // namespace

hipError_t launch_rope(const RopeArgs& args, int in_dtype, int out_dtype, hipStream_t stream) {
  RopeArgs a = args;
  const int c = a.chunk;
  const int64_t total = (int64_t)a.T * (a.Hq + a.Hk + a.Hv);
  if (c)
    while ((1 << a.gp_shift) < a.D / (2 * c)) ++a.gp_shift;
  // A wavefront to a workgroup where there are fewer than four per CU.
  const int threads = (total << a.gp_shift) < 4 * 64 * (int64_t)a.cus ? 64 : kRopeThreads;
  const void* fn = nullptr;
  if (in_dtype == out_dtype)
    fn = in_dtype == MGI_F32    ? rope_kernel<float, float>(a)
         : in_dtype == MGI_BF16 ? rope_kernel<bf16_t, bf16_t>(a)
                                : rope_kernel<f16_t, f16_t>(a);
  else if (in_dtype == MGI_F32)
    fn = out_dtype == MGI_BF16 ? rope_kernel<float, bf16_t>(a)
                               : rope_kernel<float, f16_t>(a);
  else if (out_dtype == MGI_F32)
    fn = in_dtype == MGI_BF16 ? rope_kernel<bf16_t, float>(a)
                              : rope_kernel<f16_t, float>(a);
  else
    return hipErrorInvalidValue;
  void* kargs[] = {&a};
  if (c == 0)
    return hipLaunchKernel(fn, dim3((unsigned)((total + 3) / 4)), dim3(kRopeThreads), kargs, 0, stream);
  const int64_t per = threads >> a.gp_shift;
  return hipLaunchKernel(fn, dim3((unsigned)((total + per - 1) / per)), dim3(threads), kargs, 0, stream);
}

}  // namespace mgi
