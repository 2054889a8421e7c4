// paged_shared.h -- decode attention of a batch whose sequences begin with the
// same cached blocks, for gfx950.
//
// Row b's query heads attend c_b = context_lens[b] tokens; the first P = shared * S
// of them lie in blocks that all rows share, those of table row 0:
//   out[b,h,:] = sum_t softmax_t(scale q[b,h,:] . K[t,h/G,:]) V[t,h/G,:]
// with G = Hq / Hk query heads per KV head. Every sum over tokens can be cut
// anywhere: a piece leaves its largest score m (log2 units), l = sum 2^(s - m) and
// o = sum 2^(s - m) V, and pieces join as
//   M = max m_i,  L = sum l_i 2^(m_i - M),  out = sum o_i 2^(m_i - M) / L.
// So the shared tokens are attended once for all rows together, as a matrix
// product with up to 64 query rows per wavefront, each row's own tokens by
// itself, and a second launch joins the pieces. A row shorter than P takes no part
// in the shared piece (all of its tokens are its own then), so no key of either
// kind is masked for one row and not for another.
//
// Both products run on the matrix cores, straight from registers, without LDS:
//   S^T = K Q^T   A: lane l holds 16 bytes of key l & 15; B: of query l & 15.
//                 The result leaves lane l the scores of query l & 15 with keys
//                 4 (l >> 4) + i -- which is the B operand the second needs.
//   O^T += V^T P^T  A: for head dim index m = l & 15 of each 16-wide tile, the 8
//                 keys of the lane group. A lane loads a 16-byte piece of each
//                 of its 8 keys' rows (dims 8 m .. 8 m + 7: sixteen lanes read a
//                 whole row) and transposes the 8 x 8 block with 32 v_perm_b32,
//                 tile t then standing for dims 8 m + t.
// f32 uses the 16x16x4 product, one key per lane group, and needs no transpose.
// The weights 2^(s - m) are rounded to the 16-bit type for the second product
// (half a step of each weight, which the output's own rounding exceeds); the
// sums l, the scores and the outputs are f32.
//
// The running maximum moves only when a score passes it by 2^kLazy, which costs
// one comparison per tile instead of a reduction over lanes; weights stay below
// 2^kLazy, well inside every type. A tile's K and V are loaded one tile ahead.
#pragma once

#include <type_traits>

#include "mgi_common.h"
#include "mgi_internal.h"
#include "minivllm_hip.h"

namespace mgi {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kLazy = 6.f;

template <typename T>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
  if constexpr (std::is_same_v<T, bf16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const f32x2 x = {lo, hi};
  if constexpr (std::is_same_v<T, bf16_t>) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint2& v, int i) { return i == 0 ? v.x : v.y; }
__device__ __forceinline__ float fword(const uint4& v, int i) { return __uint_as_float(word(v, i)); }
__device__ __forceinline__ float across_groups_max(float x) {
  x = fmaxf(x, swizzle_xor16(x));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float across_groups_sum(float x) {
  x += swizzle_xor16(x);
  return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Sizes of one tile: KEYS keys, held by a wavefront.
template <typename T, int DP>
struct Tile {
  static constexpr int kKeys = sizeof(T) == 2 ? 32 : 16;
  static constexpr int kGroups = kKeys / 16;            // 16-key groups
  static constexpr int kCE = 16 / (int)sizeof(T);       // elements of a 16-byte chunk
  static constexpr int kKS = DP / (4 * kCE);            // chunks of a key row per lane: (l >> 4) + 4 s
  static constexpr int kEV = DP / 16 < kCE ? DP / 16 : kCE;  // value elements per load
  static constexpr int kHF = DP / (16 * kEV);           // loads per value row
  static constexpr int kRows = kKeys / 4;               // value rows per lane: 16 (j / 4) + 4 (l >> 4) + j % 4
  static constexpr int kDT = DP / 16;                   // 16-wide tiles of the head dim
  using VVec = std::conditional_t<kEV * sizeof(T) == 16, uint4, uint2>;
  uint4 k[kGroups][kKS];
  VVec v[kRows][kHF];
  bool full;       // every key counts
  uint32_t mask;   // bit j: value row j's key counts
};

// Running softmax of NQ x 16 query rows; lane l holds row l & 15 of each.
template <int DP, int NQ>
struct State {
  f32x4 acc[NQ][DP / 16];  // O^T
  float m[NQ];             // running maximum, raw scores
  float mc[NQ];            // the same times the scale, 0 while it is -inf
  float l[NQ];             // this lane group's part of the sum
  bool any;                // some key counted
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      m[q] = kNegInf;
      mc[q] = l[q] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    any = false;
  }
};

// n / d for 0 <= n < 2^31 (see magic_of).
__device__ __forceinline__ int fast_div(int n, uint32_t mul, int shift, int d) {
  return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift);
}

// Entry j of row b's table: the shared blocks are row 0's.
__device__ __forceinline__ int64_t table_entry(const SharedArgs& a, int b, int j) {
  return load_index(a.bt, a.bt_i64, (int64_t)(j < a.shared ? 0 : b) * a.bt_sb + (int64_t)j * a.bt_sm);
}

// The pool block ids of a tile's groups, one per 16 keys (S a multiple of 16).
template <int GROUPS>
struct Ids {
  int64_t id[GROUPS];
};
template <int GROUPS>
__device__ __forceinline__ Ids<GROUPS> load_ids(const SharedArgs& a, int b, int t0, int end) {
  Ids<GROUPS> r;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int tok = t0 + 16 * g;
    r.id[g] = tok < end ? table_entry(a, b, fast_div(tok, a.s_mul, a.s_shift, a.S)) : -1;
  }
  return r;
}

// Loads the tile of keys t0 .. of one KV head. UNI: S is a multiple of 16, so a
// 16-key group lies in one block and its addresses are a scalar base and a lane
// offset; otherwise every lane looks its keys up. FULL: D == DP.
template <typename T, int DP, bool UNI, bool FULL>
__device__ __forceinline__ void load_tile(const SharedArgs& a, int b, int kvh, int t0, int end,
                                          const Ids<Tile<T, DP>::kGroups>& ids, Tile<T, DP>& f) {
  using L = Tile<T, DP>;
  const int lane = (int)threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
  const char* kp = (const char*)a.k + (int64_t)kvh * a.k_sh * (int)sizeof(T);
  const char* vp = (const char*)a.v + (int64_t)kvh * a.v_sh * (int)sizeof(T);
  const uint32_t k_ss = (uint32_t)a.k_ss * sizeof(T), v_ss = (uint32_t)a.v_ss * sizeof(T);
  const uint32_t vcol = (uint32_t)(row * L::kEV) * sizeof(T);
  using V = typename L::VVec;
  auto chunk_ok = [&](int s) { return FULL || (kg + 4 * s) * L::kCE < a.D; };
  auto col_ok = [&](int h) { return FULL || 16 * L::kEV * h + row * L::kEV < a.D; };
  if constexpr (UNI) {
    bool full = t0 + L::kKeys <= end;
    uint32_t mask = 0;
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g) {
      const int tok = t0 + 16 * g;
      int64_t id = ids.id[g];
      const bool ok = id >= 0 && id < a.N;
      full &= ok;
      id = ok ? id : 0;
      // Rows past the end read the last valid one again; its values are cleared.
      const int n = ok ? min(16, max(0, end - tok)) : 0;
      const int blk = fast_div(tok, a.s_mul, a.s_shift, a.S), off = ok ? tok - blk * a.S : 0;
      const char* kb = kp + (id * a.k_sn + (int64_t)off * a.k_ss) * (int)sizeof(T);
      const char* vb = vp + (id * a.v_sn + (int64_t)off * a.v_ss) * (int)sizeof(T);
      const int last = max(n, 1) - 1;
      const uint32_t kr = (uint32_t)min(row, last) * k_ss + (uint32_t)kg * 16;
#pragma unroll
      for (int s = 0; s < L::kKS; ++s)
        f.k[g][s] = chunk_ok(s) ? *(const uint4*)(kb + (kr + 64 * s)) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = 4 * kg + j;
        mask |= (key < n ? 1u : 0u) << (4 * g + j);
        const uint32_t vr = (uint32_t)min(key, last) * v_ss + vcol;
#pragma unroll
        for (int h = 0; h < L::kHF; ++h)
          f.v[4 * g + j][h] = col_ok(h) ? *(const V*)(vb + (vr + 16 * L::kEV * (int)sizeof(T) * h)) : V{};
      }
    }
    f.full = full;
    f.mask = mask;
  } else {
    auto find = [&](int key, bool* ok) {
      const int k = min(key, end - 1), blk = fast_div(k, a.s_mul, a.s_shift, a.S);
      const int64_t id = table_entry(a, b, blk);
      *ok = key < end && id >= 0 && id < a.N;
      return *ok ? make_longlong2(id, k - blk * a.S) : make_longlong2(0, 0);
    };
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g) {
      bool ok;
      const longlong2 at = find(t0 + 16 * g + row, &ok);
      const char* p = kp + (at.x * a.k_sn + at.y * a.k_ss) * (int)sizeof(T) + kg * 16;
#pragma unroll
      for (int s = 0; s < L::kKS; ++s) f.k[g][s] = chunk_ok(s) ? *(const uint4*)(p + 64 * s) : make_uint4(0, 0, 0, 0);
    }
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < L::kRows; ++j) {
      bool ok;
      const longlong2 at = find(t0 + 16 * (j / 4) + 4 * kg + j % 4, &ok);
      mask |= (ok ? 1u : 0u) << j;
      const char* p = vp + (at.x * a.v_sn + at.y * a.v_ss) * (int)sizeof(T) + vcol;
#pragma unroll
      for (int h = 0; h < L::kHF; ++h)
        f.v[j][h] = col_ok(h) ? *(const V*)(p + 16 * L::kEV * (int)sizeof(T) * h) : V{};
    }
    f.mask = mask;
    f.full = __all(mask == (1u << L::kRows) - 1);
  }
}

// One tile's scores, weights and products for NQ x 16 query rows.
template <typename T, int DP, int NQ>
__device__ __forceinline__ void attend_tile(const SharedArgs& a, Tile<T, DP>& f, const uint4 (&qf)[NQ][Tile<T, DP>::kKS],
                                            State<DP, NQ>& st) {
  using L = Tile<T, DP>;
  f32x4 s[NQ][L::kGroups];
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g) s[q][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < L::kKS; ++c)
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        if constexpr (sizeof(T) == 2) {
          s[q][g] = mfma16<T>(f.k[g][c], qf[q][c], s[q][g]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[q][g] = __builtin_amdgcn_mfma_f32_16x16x4f32(fword(f.k[g][c], e), fword(qf[q][c], e), s[q][g], 0, 0, 0);
        }
      }
  if (!f.full) {
#pragma unroll
    for (int j = 0; j < L::kRows; ++j) {
      const bool ok = (f.mask >> j) & 1;
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[q][j / 4][j % 4] = ok ? s[q][j / 4][j % 4] : kNegInf;
      // A weight of 0 times an infinity or NaN in an unused slot is no 0.
#pragma unroll
      for (int h = 0; h < L::kHF; ++h) f.v[j][h] = ok ? f.v[j][h] : typename L::VVec{};
    }
    st.any |= __any(f.mask != 0);
  } else {
    st.any = true;
  }
  const float c = a.scale_log2, slack = a.lazy;
  float top[NQ];
  bool moves = false;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    top[q] = kNegInf;
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[q] = fmaxf(top[q], s[q][g][i]);
    moves |= top[q] > st.m[q] + slack;
  }
  if (__any(moves)) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const float mn = fmaxf(st.m[q], across_groups_max(top[q]));
      const float mcn = mn == kNegInf ? 0.f : mn * c;
      const float alpha = st.m[q] == kNegInf ? 0.f : fast_exp2(st.mc[q] - mcn);
      st.m[q] = mn;
      st.mc[q] = mcn;
      st.l[q] *= alpha;
#pragma unroll
      for (int t = 0; t < L::kDT; ++t) st.acc[q][t] *= alpha;
    }
  }
  float p[NQ][L::kRows];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < L::kRows; ++j) {
      p[q][j] = fast_exp2(fmaf(s[q][j / 4][j % 4], c, -st.mc[q]));
      sum += p[q][j];
    }
    st.l[q] += sum;
  }
  if constexpr (sizeof(T) == 2) {
    uint4 pf[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      pf[q] = make_uint4(pack2<T>(p[q][0], p[q][1]), pack2<T>(p[q][2], p[q][3]), pack2<T>(p[q][4], p[q][5]),
                         pack2<T>(p[q][6], p[q][7]));
#pragma unroll
    for (int h = 0; h < L::kHF; ++h)
#pragma unroll
      for (int u = 0; u < L::kEV / 2; ++u)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const uint32_t sel = odd ? 0x07060302u : 0x05040100u;
          uint4 av;
          av.x = __builtin_amdgcn_perm(word(f.v[1][h], u), word(f.v[0][h], u), sel);
          av.y = __builtin_amdgcn_perm(word(f.v[3][h], u), word(f.v[2][h], u), sel);
          av.z = __builtin_amdgcn_perm(word(f.v[5][h], u), word(f.v[4][h], u), sel);
          av.w = __builtin_amdgcn_perm(word(f.v[7][h], u), word(f.v[6][h], u), sel);
          const int t = L::kEV * h + 2 * u + odd;
#pragma unroll
          for (int q = 0; q < NQ; ++q) st.acc[q][t] = mfma16<T>(av, pf[q], st.acc[q][t]);
        }
  } else {
#pragma unroll
    for (int h = 0; h < L::kHF; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            st.acc[q][4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(fword(f.v[j][h], e), p[q][j], st.acc[q][4 * h + e], 0, 0, 0);
  }
}

// Attends the tiles first, first + step, ... below end, the next one loading
// while one is computed.
template <typename T, int DP, int NQ, bool UNI, bool FULL>
__device__ __forceinline__ void stream_tiles(const SharedArgs& a, int b, int kvh, int first, int step, int end,
                                             const uint4 (&qf)[NQ][Tile<T, DP>::kKS], State<DP, NQ>& st) {
  using L = Tile<T, DP>;
  if (first >= end) return;
  L f0, f1;
  Ids<L::kGroups> ids{};
  if constexpr (UNI) ids = load_ids<L::kGroups>(a, b, first, end);
  load_tile<T, DP, UNI, FULL>(a, b, kvh, first, end, ids, f0);
  int t = first + step;
  if constexpr (UNI) ids = load_ids<L::kGroups>(a, b, t, end);
  while (true) {
    Ids<L::kGroups> next{};
    if (t < end) {
      if constexpr (UNI) next = load_ids<L::kGroups>(a, b, t + step, end);
      load_tile<T, DP, UNI, FULL>(a, b, kvh, t, end, ids, f1);
    }
    attend_tile<T, DP, NQ>(a, f0, qf, st);
    if (t >= end) break;
    t += step;
    if (t < end) {
      if constexpr (UNI) ids = load_ids<L::kGroups>(a, b, t + step, end);
      load_tile<T, DP, UNI, FULL>(a, b, kvh, t, end, next, f0);
    }
    attend_tile<T, DP, NQ>(a, f1, qf, st);
    if (t >= end) break;
    t += step;
  }
}

// Query fragments of NQ x 16 rows of one KV head's query heads: row r is sequence
// r / G's head r % G, from row r0 on; rows past `rows` are zero.
template <typename T, int DP, int NQ, bool FULL>
__device__ __forceinline__ void load_queries(const SharedArgs& a, int kvh, int64_t r0, int64_t rows,
                                             uint4 (&qf)[NQ][Tile<T, DP>::kKS]) {
  using L = Tile<T, DP>;
  const int lane = (int)threadIdx.x & 63, kg = lane >> 4;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t r = r0 + 16 * q + (lane & 15);
    const int bb = fast_div((int)r, a.g_mul, a.g_shift, a.G), g = (int)r - bb * a.G;
    const T* p = (const T*)a.q + (int64_t)bb * a.q_sb + (int64_t)(kvh * a.G + g) * a.q_sh + kg * L::kCE;
#pragma unroll
    for (int s = 0; s < L::kKS; ++s) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < rows && (FULL || (kg + 4 * s) * L::kCE < a.D)) {
        x = *(const uint4*)(p + 4 * L::kCE * s);
        x = make_uint4(x.x ^ a.q_flip, x.y ^ a.q_flip, x.z ^ a.q_flip, x.w ^ a.q_flip);
      }
      qf[q][s] = a.q_zero ? make_uint4(0, 0, 0, 0) : x;
    }
  }
}

// What a row's sum stands for in a partial: l > 0 (or NaN) with its maximum; 0 no
// key counted; -1 keys counted and every score was -inf.
__device__ __forceinline__ float coded_sum(float l, bool any) { return l == 0.f && any ? -1.f : l; }

// Joins the states of the workgroup's wavefronts into wavefront 0's: st.mc is then
// the maximum (log2 units, kNegInf for none) and st.l the coded sum.
template <int DP, int NQ, int WAVES>
__device__ __forceinline__ void join_waves(State<DP, NQ>& st, int wave, float (*ml)[2][NQ * 16], f32x4* buf) {
  const int lane = (int)threadIdx.x & 63, row = lane & 15;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    st.l[q] = coded_sum(across_groups_sum(st.l[q]), st.any);
    st.mc[q] = st.m[q] == kNegInf ? kNegInf : st.mc[q];
    if (lane < 16) {
      ml[wave][0][16 * q + row] = st.mc[q];
      ml[wave][1][16 * q + row] = st.l[q];
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    float top = kNegInf, sum = 0.f;
    bool dead = false;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ml[w][0][16 * q + row]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float m = ml[w][0][16 * q + row], l = ml[w][1][16 * q + row];
      if (l <= 0.f) dead |= l < 0.f;
      else sum += l * fast_exp2(m - top);
    }
    const float mine = st.l[q] <= 0.f ? 0.f : fast_exp2(st.mc[q] - top);
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) st.acc[q][t] *= mine;
    st.mc[q] = top;
    st.l[q] = sum == 0.f && dead ? -1.f : sum;
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int half = WAVES / 2; half > 0; half >>= 1) {
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) buf[((wave - half) * (DP / 16) + t) * 64 + lane] = st.acc[q][t];
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) st.acc[q][t] += buf[(wave * (DP / 16) + t) * 64 + lane];
      }
      __syncthreads();
    }
}

// Calls f(d, x) for the runs of kEV consecutive head dims d .. that the lane
// holds of query tile q.
template <typename T, int DP, int NQ, typename F>
__device__ __forceinline__ void each_run(const SharedArgs& a, const State<DP, NQ>& st, int q, F f) {
  using L = Tile<T, DP>;
  const int kg = ((int)threadIdx.x & 63) >> 4;
#pragma unroll
  for (int h = 0; h < L::kHF; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 16 * L::kEV * h + L::kEV * (4 * kg + i);
      float x[L::kEV];
#pragma unroll
      for (int t = 0; t < L::kEV; ++t) x[t] = st.acc[q][L::kEV * h + t][i];
      if (d < a.D) f(d, x);
    }
}

// Writes the lane's row of query tile q as the partial of slot `slot`.
template <typename T, int DP, int NQ>
__device__ __forceinline__ void store_partial(const SharedArgs& a, const State<DP, NQ>& st, int q, int64_t slot,
                                              float m, float l) {
  if (((int)threadIdx.x & 63) < 16) a.ws_ml[slot] = make_float2(m, l);
  float* row = a.ws_acc + slot * a.D;
  each_run<T>(a, st, q, [&](int d, const float* x) {
#pragma unroll
    for (int e = 0; e < Tile<T, DP>::kEV; e += 4) *(float4*)(row + d + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
  });
}

__device__ __forceinline__ int clamped_ctx(const SharedArgs& a, int b) {
  const int64_t c = load_index(a.cl, a.cl_i64, (int64_t)b * a.cl_s), top = (int64_t)a.M * a.S;
  return (int)(c < 0 ? 0 : c > top ? top : c);
}

// Row b's own tokens are first .. end - 1.
struct Own {
  int first, end;
};
__device__ __forceinline__ Own own_range(const SharedArgs& a, int b) {
  const int c = clamped_ctx(a, b);
  return {c < a.P ? 0 : a.P, c};
}

// The list of all rows' own tiles, (b, virtual head, tile) in that order, cut into
// equal segments, one per wavefront. A virtual head is a KV head and a set of at
// most 16 of its query heads.
__device__ __forceinline__ int segment_tiles(const SharedArgs& a, int total) {
  return max(a.own_min_tiles, (int)(((int64_t)total + a.own_waves - 1) / a.own_waves));
}

template <typename T, int DP, bool UNI, bool FULL>
__device__ __forceinline__ void attend_own(const SharedArgs& a, int wave_index, int* cum) {
  using L = Tile<T, DP>;
  const int lane = (int)threadIdx.x & 63;
  // cum[b]: tiles of rows 0 .. b, of one virtual head.
  const int total = uniform(cum[a.B - 1]) * a.vheads, seg = segment_tiles(a, total);
  const int64_t lo64 = (int64_t)wave_index * seg;
  if (lo64 >= total) return;
  int u = (int)lo64;
  const int stop = (int)min((int64_t)total, lo64 + seg);
  int b = 0;
  {  // the row of tile u: the first with cum[b] * vheads > u
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] * a.vheads > u) hi = mid;
      else lo = mid + 1;
    }
    b = lo;
  }
  uint4 qf[1][L::kKS];
  State<DP, 1> st;
  while (u < stop) {
    b = uniform(b);
    const int before = b ? uniform(cum[b - 1]) : 0, tiles = uniform(cum[b]) - before;
    if (tiles == 0) {
      ++b;
      continue;
    }
    const int rem = u - before * a.vheads;
    const int vh = rem / tiles, tile = rem - vh * tiles;
    const int n = min(tiles - tile, stop - u);
    const int kvh = vh / a.gsets, g0 = (vh - kvh * a.gsets) * 16;
    const Own own = own_range(a, b);
    load_queries<T, DP, 1, FULL>(a, kvh, (int64_t)b * a.G + g0, (int64_t)(b + 1) * a.G, qf);
    st.reset();
    const int first = own.first + tile * L::kKeys;
    stream_tiles<T, DP, 1, UNI, FULL>(a, b, kvh, first, L::kKeys, min(own.end, first + n * L::kKeys), qf, st);
    const int g = g0 + (lane & 15);
    const float l = coded_sum(across_groups_sum(st.l[0]), st.any);
    // A piece that begins its row's tiles has the row's slot, another the segment's.
    const int64_t slot = tile == 0 ? a.own_slot + (int64_t)b * a.Hq + kvh * a.G + g
                                   : a.cont_slot + (int64_t)wave_index * 16 + (lane & 15);
    if (g < a.G) store_partial<T>(a, st, 0, slot, st.m[0] == kNegInf ? kNegInf : st.mc[0], l);
    u += n;
    if (vh == a.vheads - 1 && tile + n == tiles) ++b;
  }
}

constexpr int kSplitWaves = 4;

// The pieces: workgroups 0 .. prefix_wgs - 1 take the shared tokens, (KV head,
// query rows, range of tokens) each; the wavefronts of the others the rows' own.
template <typename T, int DP, int NQ, bool UNI, bool FULL>
__global__ void __launch_bounds__(64 * kSplitWaves) paged_shared_split(const SharedArgs a) {
  using L = Tile<T, DP>;
  __shared__ __align__(16) char lds[kSplitWaves / 2 * (DP / 16) * 64 * 16 > kSharedMaxB * 4
                                        ? kSplitWaves / 2 * (DP / 16) * 64 * 16 : kSharedMaxB * 4];
  __shared__ float ml[kSplitWaves][2][NQ * 16];
  __shared__ int part[kSplitWaves];
  const int wave = uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  if ((int)blockIdx.x < a.prefix_wgs) {
    const int i = (int)blockIdx.x, rest = i / a.row_sets, set = i - rest * a.row_sets;
    const int kvh = rest / a.chunks, chunk = rest - kvh * a.chunks;
    const int64_t rows = (int64_t)a.B * a.G, r0 = (int64_t)set * 16 * NQ;
    int slot_b[NQ], slot_g[NQ];
    bool takes[NQ], some = false;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int r = (int)r0 + 16 * q + (lane & 15);
      slot_b[q] = fast_div(r, a.g_mul, a.g_shift, a.G);
      slot_g[q] = r - slot_b[q] * a.G;
      takes[q] = r < rows && clamped_ctx(a, slot_b[q]) >= a.P;
      some |= takes[q];
    }
    if (!__any(some)) return;  // the same in every wavefront of the workgroup
    uint4 qf[NQ][L::kKS];
    State<DP, NQ> st;
    load_queries<T, DP, NQ, FULL>(a, kvh, r0, rows, qf);
    st.reset();
    const int first = chunk * a.chunk_tiles * L::kKeys, end = min(a.P, first + a.chunk_tiles * L::kKeys);
    stream_tiles<T, DP, NQ, UNI, FULL>(a, 0, kvh, first + wave * L::kKeys, kSplitWaves * L::kKeys, end, qf, st);
    join_waves<DP, NQ, kSplitWaves>(st, wave, ml, (f32x4*)lds);
    if (wave == 0) {
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        if (takes[q])
          store_partial<T>(a, st, q, ((int64_t)slot_b[q] * a.Hq + kvh * a.G + slot_g[q]) * a.chunks + chunk, st.mc[q], st.l[q]);
    }
    return;
  }
  // Prefix sums of the rows' own tiles, in LDS; the first of these workgroups
  // leaves them for the joining launch.
  int* cum = (int*)lds;
  const int per = (a.B + 64 * kSplitWaves - 1) / (64 * kSplitWaves), b0 = (int)threadIdx.x * per;
  int sum = 0;
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    if (b < a.B) {
      const Own own = own_range(a, b);
      sum += (own.end - own.first + L::kKeys - 1) / L::kKeys;
      cum[b] = sum;
    }
  }
  int incl = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(incl, d, 64);
    if (lane >= d) incl += y;
  }
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int base = incl - sum;
  for (int w = 0; w < wave; ++w) base += part[w];
  for (int i = 0; i < per; ++i)
    if (b0 + i < a.B) {
      const int v = cum[b0 + i] + base;
      cum[b0 + i] = v;
      if ((int)blockIdx.x == a.prefix_wgs) a.ws_cum[b0 + i] = v;
    }
  __syncthreads();
  const int wave_index = ((int)blockIdx.x - a.prefix_wgs) * kSplitWaves + wave;
  attend_own<T, DP, UNI, FULL>(a, wave_index, cum);
}

// Joins the partials of one (row, query head) per wavefront.
template <typename T>
__global__ void __launch_bounds__(256) paged_shared_join(const SharedArgs a) {
  const int lane = (int)threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);
  if (unit >= (int64_t)a.B * a.Hq) return;
  const int b = (int)(unit / a.Hq), hq = (int)(unit - (int64_t)b * a.Hq);
  const int kvh = hq / a.G, g = hq - kvh * a.G, set = g / 16;
  const int before = b ? a.ws_cum[b - 1] : 0, tiles = a.ws_cum[b] - before;
  const int seg = segment_tiles(a, a.ws_cum[a.B - 1] * a.vheads);
  const int u = before * a.vheads + (kvh * a.gsets + set) * tiles;
  const int w0 = u / seg, pieces = tiles ? (u + tiles - 1) / seg - w0 + 1 : 0;
  const int shared = clamped_ctx(a, b) >= a.P ? a.chunks : 0, n = shared + pieces;
  auto slot = [&](int i) -> int64_t {
    if (i < shared) return unit * a.chunks + i;
    if (i == shared) return a.own_slot + unit;
    return a.cont_slot + (int64_t)(w0 + i - shared) * 16 + (g - set * 16);
  };
  float top = kNegInf;
  for (int i = lane; i < n; i += 64) {
    const float2 x = a.ws_ml[slot(i)];
    if (!(x.y <= 0.f)) top = fmaxf(top, x.x);
  }
  top = wave_max(top);
  float sum = 0.f;
  bool dead = false;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < n; ++i) {
    const int64_t s = slot(i);
    const float2 x = a.ws_ml[s];
    if (x.y <= 0.f) {
      dead |= x.y < 0.f;
      continue;
    }
    const float w = fast_exp2(x.x - top);
    sum += x.y * w;
    if (4 * lane < a.D) acc += w * *(const f32x4*)(a.ws_acc + s * a.D + 4 * lane);
  }
  const float r = sum == 0.f ? (dead ? __builtin_nanf("") : 0.f) : 1.f / sum;
  if (4 * lane < a.D) {
    T* o = (T*)a.out + (int64_t)b * a.o_sb + (int64_t)hq * a.o_sh + 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e) Elem<T>::store(o + e, acc[e] * r);
  }
}

// One workgroup per (row, virtual head): all of the row's tokens in one launch.
template <int DP>
constexpr int kOneWaves = DP > 128 ? 4 : 8;
template <typename T, int DP, bool UNI, bool FULL>
__global__ void __launch_bounds__(64 * kOneWaves<DP>) paged_shared_one(const SharedArgs a) {
  using L = Tile<T, DP>;
  __shared__ f32x4 buf[kOneWaves<DP> / 2 * (DP / 16) * 64];
  __shared__ float ml[kOneWaves<DP>][2][16];
  const int wave = uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int b = (int)blockIdx.y, vh = (int)blockIdx.x, kvh = vh / a.gsets, g0 = (vh - kvh * a.gsets) * 16;
  const int end = clamped_ctx(a, b);
  uint4 qf[1][L::kKS];
  State<DP, 1> st;
  load_queries<T, DP, 1, FULL>(a, kvh, (int64_t)b * a.G + g0, (int64_t)(b + 1) * a.G, qf);
  st.reset();
  stream_tiles<T, DP, 1, UNI, FULL>(a, b, kvh, wave * L::kKeys, kOneWaves<DP> * L::kKeys, end, qf, st);
  join_waves<DP, 1, kOneWaves<DP>>(st, wave, ml, buf);
  const int g = g0 + (lane & 15);
  if (wave || g >= a.G) return;
  const float r = st.l[0] == 0.f ? 0.f : st.l[0] < 0.f ? __builtin_nanf("") : 1.f / st.l[0];
  T* o = (T*)a.out + (int64_t)b * a.o_sb + (int64_t)(kvh * a.G + g) * a.o_sh;
  each_run<T>(a, st, 0, [&](int d, const float* x) {
#pragma unroll
    for (int e = 0; e < L::kEV; ++e) Elem<T>::store(o + d + e, x[e] * r);
  });
}

// Any strides, any head_dim up to 512: one wavefront per (row, query head), token
// by token.
template <typename T>
__global__ void __launch_bounds__(64) paged_shared_any(const SharedArgs a) {
  const int lane = (int)threadIdx.x, b = (int)blockIdx.y, hq = (int)blockIdx.x, kvh = hq / a.G;
  const int n = clamped_ctx(a, b);
  const T* q = (const T*)a.q + (int64_t)b * a.q_sb + (int64_t)hq * a.q_sh;
  float x[8], acc[8], m = kNegInf, l = 0.f;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 64 * i;
    x[i] = d < a.D && !a.q_zero ? Elem<T>::load(q + (int64_t)d * a.q_sd) : 0.f;
    if (a.q_flip) x[i] = -x[i];
    acc[i] = 0.f;
  }
  int64_t id = -1;
  for (int t = 0; t < n; ++t) {
    const int blk = t / a.S, off = t - blk * a.S;
    if (off == 0) id = table_entry(a, b, blk);
    if (id < 0 || id >= a.N) continue;
    any = true;
    const T* k = (const T*)a.k + id * a.k_sn + off * a.k_ss + (int64_t)kvh * a.k_sh;
    const T* v = (const T*)a.v + id * a.v_sn + off * a.v_ss + (int64_t)kvh * a.v_sh;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 64 * i;
      if (d < a.D) s = fmaf(x[i], Elem<T>::load(k + (int64_t)d * a.k_sd), s);
    }
    s = wave_sum(s) * a.scale_log2;
    const float mn = fmaxf(m, s), safe = mn == kNegInf ? 0.f : mn;
    const float alpha = m == kNegInf ? 0.f : fast_exp2(m - safe), p = fast_exp2(s - safe);
    m = mn;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 64 * i;
      if (d < a.D) acc[i] = fmaf(p, Elem<T>::load(v + (int64_t)d * a.v_sd), acc[i] * alpha);
    }
  }
  const float r = l == 0.f ? (any ? __builtin_nanf("") : 0.f) : 1.f / l;
  T* o = (T*)a.out + (int64_t)b * a.o_sb + (int64_t)hq * a.o_sh;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 64 * i;
    if (d < a.D) Elem<T>::store(o + (int64_t)d * a.o_sd, acc[i] * r);
  }
}

template <typename T, int DP, bool UNI, bool FULL>
hipError_t launch_tiles(const SharedArgs& a, hipStream_t stream) {
  SharedArgs c = a;
  void* kargs[] = {&c};
  if (a.one_launch)
    return hipLaunchKernel((const void*)&paged_shared_one<T, DP, UNI, FULL>, dim3((unsigned)a.vheads, (unsigned)a.B),
                           dim3(64 * kOneWaves<DP>), kargs, 0, stream);
  const void* fn = (const void*)&paged_shared_split<T, DP, 1, UNI, FULL>;
  if (a.row_tiles == 2) fn = (const void*)&paged_shared_split<T, DP, 2, UNI, FULL>;
  if constexpr (DP < 256)
    if (a.row_tiles == 4) fn = (const void*)&paged_shared_split<T, DP, 4, UNI, FULL>;
  const unsigned wgs = (unsigned)(a.prefix_wgs + a.own_waves / kSplitWaves);
  const hipError_t e = hipLaunchKernel(fn, dim3(wgs), dim3(64 * kSplitWaves), kargs, 0, stream);
  if (e != hipSuccess) return e;
  const int64_t units = (int64_t)a.B * a.Hq;
  return hipLaunchKernel((const void*)&paged_shared_join<T>, dim3((unsigned)((units + 3) / 4)), dim3(256), kargs, 0, stream);
}

template <typename T, int DP>
hipError_t launch_width(const SharedArgs& a, hipStream_t stream) {
  if (a.S % 16 != 0) return launch_tiles<T, DP, false, false>(a, stream);
  return a.D == DP ? launch_tiles<T, DP, true, true>(a, stream) : launch_tiles<T, DP, true, false>(a, stream);
}

template <typename T>
hipError_t launch_type(const SharedArgs& a, hipStream_t stream) {
  if (!a.tiles) {
    SharedArgs c = a;
    void* kargs[] = {&c};
    return hipLaunchKernel((const void*)&paged_shared_any<T>, dim3((unsigned)a.Hq, (unsigned)a.B), dim3(64), kargs, 0, stream);
  }
  return a.D <= 64 ? launch_width<T, 64>(a, stream) : a.D <= 128 ? launch_width<T, 128>(a, stream) : launch_width<T, 256>(a, stream);
}

}  // namespace

}  // namespace mgi
