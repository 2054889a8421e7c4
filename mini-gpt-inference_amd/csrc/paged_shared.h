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
// So the shared tokens are attended once for all rows together, as one matrix
// product, each row's own tokens by themselves, and a second launch joins the
// pieces. A row shorter than P takes no part in the shared piece (all of its tokens
// are its own then), so no key of either kind is masked for one row and not for
// another.
//
// Both products run on the matrix cores. In the register form, without LDS:
//   S^T = K Q^T   A: lane l holds 16 bytes of key l & 15; B: of query l & 15.
//                 The result leaves lane l the scores of query l & 15 with keys
//                 4 (l >> 4) + i -- which is the B operand the second needs.
//   O^T += V^T P^T  A: for head dim index m = l & 15 of each 16-wide tile, the 8
//                 keys of the lane group. A lane loads a 16-byte piece of each
//                 of its 8 keys' rows (dims 8 m .. 8 m + 7: sixteen lanes read a
//                 whole row) and transposes the 8 x 8 block with 32 v_perm_b32,
//                 tile t then standing for dims 8 m + t.
// f32 uses the 16x16x4 product, one key per lane group, and needs no transpose.
// A row's own tokens take it with one query head's row in 16 filled, or G of them:
// the products are idle lanes then, but 16 KiB of K and V take a CU 650 ns of its
// share of HBM and a wavefront's products 110 ns. Many rows on the shared tokens
// take tiles in LDS instead (below).
//
// Rounding: the weights 2^(s - m) go to the 16-bit type for the second product, at
// most half a step of each, as independent errors about as much in the output as
// its own rounding (bf16: 0.0023 off 64 bits, relative, where rounding alone is
// 0.0017; f16 0.00027 and 0.00021). f16 holds that down to 2^-14 only, so its weights
// are 2^(s - m + 13) (the sums' too, so that it divides out): half a step down to 2^-27
// of the largest, 2^-38 of it below. Scores, sums l and outputs are f32; l sums the
// weights before their rounding in the register form, the rounded ones in LDS's.
//
// The running maximum moves only when a score passes it by kSharedLazy (f16:
// kSharedLazyF16) in log2 units, which costs one comparison per tile instead of a
// reduction over lanes; weights stay inside every type.
//
// What bounds it (MI355X; inputs from memory, another set each call): 64 x 32 heads
// on 4096 shared tokens and 64-1024 of their own, bf16, 649 MB: 116 us, 5.6 TB/s; 128
// x 32 on 8 KV heads over 65 536 shared, 138 GFLOP: 172 us, 800 TFLOP/s, the softmax's
// VALU work in line with the products (37 % of cycles in the matrix cores, LDS conflicts
// none; with all keys in L2 it still takes 141 of the 146 us without own tokens).
// Calls under about 30 us are chains: launch and the rows' prefix sums 4 us, a first
// tile 3, the joining launch 5-7 us.
#pragma once

#include <type_traits>

#include "lds_tiles.h"
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

template <typename T>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
  if constexpr (std::is_same_v<T, bf16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const f32x2 x = {lo, hi};
  if constexpr (std::is_same_v<T, bf16_t>) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
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

// What the exponents of weights are taken from, in log2 units, for a maximum m (raw): m c,
// for f16 lowered by its scale. Scores past 2^20, whose product with c is off by a
// sixteenth and more, keep it as it is: the scale leaves them no room for that.
template <typename T>
__device__ __forceinline__ float exponent_base(float m, float c) {
  if (m == kNegInf) return 0.f;
  if constexpr (std::is_same_v<T, f16_t>) return fabsf(m * c) < 0x1p20f ? fmaf(m, c, -kSharedF16Scale) : m * c;
  else return m * c;
}

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
  int n[kGroups];  // S a multiple of 16: keys of each group that count
  uint32_t mask;   // other S: bit j, the lane's value row j counts
};

// Running softmax of NQ x 16 query rows; lane l holds row l & 15 of each.
template <int DP, int NQ>
struct State {
  f32x4 acc[NQ][DP / 16];  // O^T
  float m[NQ];             // running maximum, raw scores
  float mc[NQ];            // its exponent_base, 0 while it is -inf
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

// Entry j of row b's table: the shared blocks are row 0's.
__device__ __forceinline__ int64_t table_entry(const SharedArgs& a, int b, int j) {
  return load_index(a.bt, a.bt_i64, (int64_t)(j < a.shared ? 0 : b) * a.bt_sb + (int64_t)j * a.bt_sm);
}

// Where the 16-key groups of a wavefront's next tiles lie (S a multiple of 16, so
// each lies in one block): lane i holds group i % GR of tile i / GR, as byte offsets
// into the pool, and how many of its keys count. One table load serves 64 / GR tiles,
// and the next window's is issued a window ahead: an entry read where it is used
// costs a wait for every load in flight.
struct Window {
  uint32_t k_lo, k_hi, v_lo, v_hi;
  int n;
};

// The lane's table entry, as loaded, for its group, whose first token is tok. Entries
// past a row's length are read too (and not used), so that the load does not wait for
// the length; past the table its last one stands in, as a load under a condition is
// waited for where the condition ends, with all others in flight.
__device__ __forceinline__ Index window_entry(const SharedArgs& a, int b, int tok) {
  const int j = fast_div(min(tok, a.M * a.S - 1), a.s_mul, a.s_shift, a.S);
  Index x;
  x.load(a.bt, a.bt_i64, (uint64_t)(j < a.shared ? 0 : b) * (uint64_t)a.bt_sb + (uint64_t)j * (uint64_t)a.bt_sm);
  return x;
}
// The entry's block, -1 for none or one outside the pool.
__device__ __forceinline__ int entry_block(const SharedArgs& a, const Index& x, int tok) {
  const int64_t id = x.value(a.bt_i64);
  return tok < a.M * a.S && id >= 0 && id < a.N ? (int)id : -1;
}
template <typename T>
__device__ __forceinline__ Window make_window(const SharedArgs& a, int id, int tok, int end, int kvh) {
  const int64_t at = max(id, 0), off = id < 0 ? 0 : tok - fast_div(tok, a.s_mul, a.s_shift, a.S) * a.S;
  const uint64_t k = (uint64_t)(at * a.k_sn + off * a.k_ss + kvh * a.k_sh) * sizeof(T);
  const uint64_t v = (uint64_t)(at * a.v_sn + off * a.v_ss + kvh * a.v_sh) * sizeof(T);
  return {(uint32_t)k, (uint32_t)(k >> 32), (uint32_t)v, (uint32_t)(v >> 32), id < 0 ? 0 : max(0, min(16, end - tok))};
}
__device__ __forceinline__ int64_t lane_offset(uint32_t lo, uint32_t hi, int i) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)lo, i) |
                   ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, i) << 32));
}

// 16 or 8 bytes.
template <bool NT, typename V>
__device__ __forceinline__ V load_piece(const char* p) {
  if constexpr (!NT) return *(const V*)p;
  typedef uint32_t u4 __attribute__((ext_vector_type(sizeof(V) / 4)));
  return __builtin_bit_cast(V, __builtin_nontemporal_load((const u4*)p));
}

// Loads the keys, and the values, of the tile whose groups are lanes at .. of the
// window (kp, vp: the pools). Rows past a group's last key read that one again, chunks
// past D zeros: no load is under a condition. FULL: D == DP.
template <typename T, int DP, bool FULL, bool NT = false>
__device__ __forceinline__ void load_keys(const SharedArgs& a, const char* kp, const Window& w, int at, Tile<T, DP>& f) {
  using L = Tile<T, DP>;
  const int lane = (int)threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
  const uint32_t ss = (uint32_t)a.k_ss * sizeof(T);
#pragma unroll
  for (int g = 0; g < L::kGroups; ++g) {
    const int n = __builtin_amdgcn_readlane(w.n, at + g);
    const char* base = kp + lane_offset(w.k_lo, w.k_hi, at + g);
    const uint32_t off = (uint32_t)min(row, max(n, 1) - 1) * ss + (uint32_t)kg * 16;
#pragma unroll
    for (int s = 0; s < L::kKS; ++s) {
      if constexpr (FULL) {
        f.k[g][s] = load_piece<NT, uint4>(base + off + 64 * s);
      } else {
        const bool in = (kg + 4 * s) * L::kCE < a.D;
        f.k[g][s] = load_piece<NT, uint4>(in ? base + off + 64 * s : (const char*)kZeroRow);
      }
    }
  }
}
template <typename T, int DP, bool FULL, bool NT = false>
__device__ __forceinline__ void load_values(const SharedArgs& a, const char* vp, const Window& w, int at,
                                            Tile<T, DP>& f) {
  using L = Tile<T, DP>;
  using V = typename L::VVec;
  const int lane = (int)threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
  const uint32_t ss = (uint32_t)a.v_ss * sizeof(T), col = (uint32_t)(row * L::kEV) * sizeof(T);
  f.full = true;
#pragma unroll
  for (int g = 0; g < L::kGroups; ++g) {
    const int n = __builtin_amdgcn_readlane(w.n, at + g);
    const char* base = vp + lane_offset(w.v_lo, w.v_hi, at + g);
    f.n[g] = n;
    f.full &= n == 16;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t off = (uint32_t)min(4 * kg + j, max(n, 1) - 1) * ss + col;
#pragma unroll
      for (int h = 0; h < L::kHF; ++h) {
        // Dims past D load the row's first ones and are not stored.
        const bool in = FULL || 16 * L::kEV * h + row * L::kEV < a.D;
        f.v[4 * g + j][h] = load_piece<NT, V>(base + (in ? off + 16 * L::kEV * (uint32_t)sizeof(T) * h : off - col));
      }
    }
  }
}

// The same for any S: every lane looks its keys up. Keys t0 .. below end.
struct Found {
  int64_t block;
  int off;
  bool ok;
};
__device__ __forceinline__ Found find_key(const SharedArgs& a, int b, int key, int end) {
  const int k = min(key, end - 1), blk = fast_div(k, a.s_mul, a.s_shift, a.S);
  const int64_t id = table_entry(a, b, blk);
  const bool ok = key < end && id >= 0 && id < a.N;
  return {ok ? id : 0, ok ? k - blk * a.S : 0, ok};
}
template <typename T, int DP>
__device__ __forceinline__ void load_keys_any(const SharedArgs& a, const char* kp, int b, int t0, int end,
                                              Tile<T, DP>& f) {
  using L = Tile<T, DP>;
  const int lane = (int)threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
#pragma unroll
  for (int g = 0; g < L::kGroups; ++g) {
    const Found at = find_key(a, b, t0 + 16 * g + row, end);
    const char* p = kp + (at.block * a.k_sn + at.off * a.k_ss) * (int)sizeof(T) + kg * 16;
#pragma unroll
    for (int s = 0; s < L::kKS; ++s)
      f.k[g][s] = (kg + 4 * s) * L::kCE < a.D ? *(const uint4*)(p + 64 * s) : make_uint4(0, 0, 0, 0);
  }
}
template <typename T, int DP>
__device__ __forceinline__ void load_values_any(const SharedArgs& a, const char* vp, int b, int t0, int end,
                                                Tile<T, DP>& f) {
  using L = Tile<T, DP>;
  using V = typename L::VVec;
  const int lane = (int)threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
  f.mask = 0;
#pragma unroll
  for (int j = 0; j < L::kRows; ++j) {
    const Found at = find_key(a, b, t0 + 16 * (j / 4) + 4 * kg + j % 4, end);
    f.mask |= (at.ok ? 1u : 0u) << j;
    const char* p = vp + (at.block * a.v_sn + at.off * a.v_ss) * (int)sizeof(T) + row * L::kEV * (int)sizeof(T);
#pragma unroll
    for (int h = 0; h < L::kHF; ++h)
      f.v[j][h] = 16 * L::kEV * h + row * L::kEV < a.D ? *(const V*)(p + 16 * L::kEV * (int)sizeof(T) * h) : V{};
  }
  f.full = __all(f.mask == (1u << L::kRows) - 1);
}

// Scores of a tile for NQ x 16 query rows.
template <typename T, int DP, int NQ>
__device__ __forceinline__ void score_tile(const Tile<T, DP>& f, const uint4 (&qf)[NQ][Tile<T, DP>::kKS],
                                           f32x4 (&s)[NQ][Tile<T, DP>::kGroups]) {
  using L = Tile<T, DP>;
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
}

// Their weights, and the products with the values.
template <typename T, int DP, int NQ, bool UNI>
__device__ __forceinline__ void attend_tile(const SharedArgs& a, Tile<T, DP>& f, f32x4 (&s)[NQ][Tile<T, DP>::kGroups],
                                            State<DP, NQ>& st) {
  using L = Tile<T, DP>;
  if (!f.full) {
    const int kg = ((int)threadIdx.x & 63) >> 4;
    bool some = false;
#pragma unroll
    for (int j = 0; j < L::kRows; ++j) {
      const bool ok = UNI ? 4 * kg + j % 4 < f.n[j / 4] : (f.mask >> j) & 1;
      some |= ok;
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[q][j / 4][j % 4] = ok ? s[q][j / 4][j % 4] : kNegInf;
      // A weight of 0 times an infinity or NaN in an unused slot is no 0.
#pragma unroll
      for (int h = 0; h < L::kHF; ++h) f.v[j][h] = ok ? f.v[j][h] : typename L::VVec{};
    }
    st.any |= __any(some);
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
      const float mcn = exponent_base<T>(mn, c);
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
            st.acc[q][4 * h + e] =
                __builtin_amdgcn_mfma_f32_16x16x4f32(fword(f.v[j][h], e), p[q][j], st.acc[q][4 * h + e], 0, 0, 0);
  }
}

// A scale that is not positive, put into the queries (apart from their loads: it waits
// for them).
template <int NQ, int KS>
__device__ __forceinline__ void sign_queries(const SharedArgs& a, uint4 (&qf)[NQ][KS]) {
  if (!(a.q_flip | a.q_zero)) return;
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 x = qf[q][s];
      qf[q][s] = a.q_zero ? make_uint4(0, 0, 0, 0)
                          : make_uint4(x.x ^ a.q_flip, x.y ^ a.q_flip, x.z ^ a.q_flip, x.w ^ a.q_flip);
    }
}

// Row b's length, from the load and its value.
__device__ __forceinline__ Index ctx_load(const SharedArgs& a, int b) {
  Index x;
  x.load(a.cl, a.cl_i64, (uint64_t)b * (uint64_t)a.cl_s);
  return x;
}
__device__ __forceinline__ int ctx_value(const SharedArgs& a, const Index& x) {
  const int64_t c = x.value(a.cl_i64), top = (int64_t)a.M * a.S;
  return (int)(c < 0 ? 0 : c > top ? top : c);
}
__device__ __forceinline__ int clamped_ctx(const SharedArgs& a, int b) { return ctx_value(a, ctx_load(a, b)); }

// Attends the tiles first, first + step, ... below end_of() of row b's table. A tile's
// keys are loaded into the registers the one before has given its scores from, and
// its values where that one's products have been taken: half a tile is always on
// its way. (A second set of registers, a whole tile ahead, changed no call's time.)
template <typename T, int DP, int NQ, bool UNI, bool FULL, typename End>
__device__ __forceinline__ void stream_tiles(const SharedArgs& a, int b, int kvh, int first, int step, End end_of,
                                             uint4 (&qf)[NQ][Tile<T, DP>::kKS], State<DP, NQ>& st) {
  using L = Tile<T, DP>;
  const char* kp = (const char*)a.k + (int64_t)kvh * a.k_sh * (int)sizeof(T);
  const char* vp = (const char*)a.v + (int64_t)kvh * a.v_sh * (int)sizeof(T);
  constexpr int kSpan = 64 / L::kGroups;  // tiles of a window
  const int lane = (int)threadIdx.x & 63;
  int tok = 0;  // the lane's group of the next window
  Index entry = {0, 0};
  Window win{};
  if constexpr (UNI) {
    tok = first + lane / L::kGroups * step + 16 * (lane % L::kGroups);
    entry = window_entry(a, b, tok);
  }
  __builtin_amdgcn_sched_barrier(0);
  const int end = uniform(end_of());
  if (first >= end) return;
  L f;
  auto keys = [&](int i) {
    if constexpr (UNI) {
      if (i % kSpan == 0) {
        win = make_window<T>(a, entry_block(a, entry, tok), tok, end, kvh);
        tok += kSpan * step;
        entry = window_entry(a, b, tok);
      }
      load_keys<T, DP, FULL>(a, (const char*)a.k, win, i % kSpan * L::kGroups, f);
    } else {
      load_keys_any<T, DP>(a, kp, b, first + i * step, end, f);
    }
  };
  auto values = [&](int i) {
    if constexpr (UNI) load_values<T, DP, FULL>(a, (const char*)a.v, win, i % kSpan * L::kGroups, f);
    else load_values_any<T, DP>(a, vp, b, first + i * step, end, f);
  };
  const int n = (end - first + step - 1) / step;
  f32x4 s[NQ][L::kGroups];
  keys(0);
  __builtin_amdgcn_sched_barrier(0);  // keys before values, as in the loop: their wait leaves the values in flight
  values(0);
  __builtin_amdgcn_sched_barrier(0);
  sign_queries(a, qf);
  for (int i = 0; i + 1 < n; ++i) {
    score_tile<T, DP, NQ>(f, qf, s);
    keys(i + 1);
    attend_tile<T, DP, NQ, UNI>(a, f, s, st);
    values(i + 1);
  }
  score_tile<T, DP, NQ>(f, qf, s);  // the last apart: loads under no condition in the loop
  attend_tile<T, DP, NQ, UNI>(a, f, s, st);
}

// Query fragments of NQ x 16 rows of one KV head's query heads: row r is sequence
// r / G's head r % G, from row r0 on; past `rows` the last one again (and not stored).
template <typename T, int DP, int NQ, bool FULL>
__device__ __forceinline__ void load_queries(const SharedArgs& a, int kvh, int r0, int rows,
                                             uint4 (&qf)[NQ][Tile<T, DP>::kKS]) {
  using L = Tile<T, DP>;
  const int lane = (int)threadIdx.x & 63, kg = lane >> 4;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int r = min(r0 + 16 * q + (lane & 15), rows - 1), bb = fast_div(r, a.g_mul, a.g_shift, a.G), g = r - bb * a.G;
    const T* p = (const T*)a.q + (int64_t)bb * a.q_sb + (int64_t)(kvh * a.G + g) * a.q_sh + kg * L::kCE;
#pragma unroll
    for (int s = 0; s < L::kKS; ++s) {
      if constexpr (FULL) qf[q][s] = *(const uint4*)(p + 4 * L::kCE * s);
      else qf[q][s] = *((kg + 4 * s) * L::kCE < a.D ? (const uint4*)(p + 4 * L::kCE * s) : (const uint4*)kZeroRow);
    }
  }
}

// What a row's sum stands for in a partial: l > 0 (or NaN) with its maximum; 0 no
// key counted; -1 keys counted and every score was -inf.
__device__ __forceinline__ float coded_sum(float l, bool any) { return l == 0.f && any ? -1.f : l; }

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

// Joins the states of the workgroup's wavefronts: each leaves its own in LDS, and after
// one barrier every thread joins the pieces of some (row, 4 head dims) and calls
// f(row, d, o, m, l) with the unscaled output, the maximum (log2 units, kNegInf for
// none) and the coded sum. `rows` of the NQ x 16 are of interest.
template <int DP, int NQ, int WAVES>
struct JoinSpace {
  float acc[WAVES][NQ * 16][DP + 4], m[WAVES][NQ * 16], l[WAVES][NQ * 16];
  int64_t slot[NQ * 16];  // of the rows' partials, where the workgroup leaves any
};
template <typename T, int DP, int NQ, int WAVES, typename F>
__device__ __forceinline__ void join_waves(const SharedArgs& a, const State<DP, NQ>& st, int wave, int rows,
                                           JoinSpace<DP, NQ, WAVES>& space, F f) {
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int row = 16 * q + (lane & 15);
    const float l = coded_sum(across_groups_sum(st.l[q]), st.any);
    if (row >= rows) continue;
    if (lane < 16) {
      space.m[wave][row] = st.m[q] == kNegInf ? kNegInf : st.mc[q];
      space.l[wave][row] = l;
    }
    each_run<T>(a, st, q, [&](int d, const float* x) {
#pragma unroll
      for (int e = 0; e < Tile<T, DP>::kEV; e += 4)
        *(f32x4*)&space.acc[wave][row][d + e] = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
    });
  }
  __syncthreads();
  for (int i = (int)threadIdx.x; i < rows * (DP / 4); i += 64 * WAVES) {
    const int row = i / (DP / 4), d = 4 * (i - row * (DP / 4));
    if (d >= a.D) continue;
    float top = kNegInf, sum = 0.f;
    bool dead = false;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, space.m[w][row]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float l = space.l[w][row];
      dead |= l < 0.f;
      const float scale = l <= 0.f ? 0.f : fast_exp2(space.m[w][row] - top);
      if (l <= 0.f) continue;
      sum += l * scale;
      o += scale * *(const f32x4*)&space.acc[w][row][d];
    }
    f(row, d, o, top, sum == 0.f && dead ? -1.f : sum);
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
    for (int e = 0; e < Tile<T, DP>::kEV; e += 4)
      *(f32x4*)(row + d + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
  });
}

constexpr int kSplitWaves = 4;

// The work is two lists: the shared tokens' tiles, (KV head, block of row sets, tile)
// in that order, each for a team of workgroups, one to a set of query rows, that
// walk the same keys together and find them in their XCD's L2 (4 sets of 128 rows
// over 65 536 tokens: 197 us with a list per set, 173 so); and the rows' own, (row,
// virtual head, tile), a virtual head being a KV head and a set of at most 16 of its
// query heads. The launch's workgroups are dealt out between the lists by cost, and
// each list is cut into equal segments: one per team of the first, one per wavefront
// of the second. A segment's first piece may continue a run that another began: it
// leaves its partial in the segment's slots, a piece that begins a run in its row's.
struct Split {
  int shared_wgs;  // workgroups of the first list, whole teams
  int seg_shared;  // tiles of a team's segment
  int seg_own;
};
__device__ __forceinline__ Split make_split(const SharedArgs& a, int own_total) {
  const int total = a.s_units * a.s_tiles;
  const int64_t cs = ((int64_t)total * a.s_cost + (int64_t)a.s_units * a.s_piece) * a.team, co = own_total;
  Split r{};
  int teams = 0;
  if (total) {
    const int64_t fair = (a.wgs * cs + (cs + co) * a.team / 2) / ((cs + co) * a.team);
    teams = (int)max((int64_t)1, min(fair, (int64_t)(a.wgs - (own_total > 0)) / a.team));
    r.seg_shared = (total + teams - 1) / teams;
  }
  r.shared_wgs = teams * a.team;
  const int waves = (a.wgs - r.shared_wgs) * kSplitWaves;
  if (waves) r.seg_own = max(1, (own_total + waves - 1) / waves);
  return r;
}

// Workgroup blockIdx.x's place: XCD blockIdx.x % 8 takes a contiguous run of each
// list (sets of rows that read the same keys then share its L2), and starts with
// its part of the first.
struct Place {
  bool shared;
  int index;  // in its list's workgroups
};
__device__ __forceinline__ Place make_place(const SharedArgs& a, const Split& sp) {
  const int x = (int)blockIdx.x & 7, j = (int)blockIdx.x >> 3;
  const int each = sp.shared_wgs / 8, rest = sp.shared_wgs % 8;
  const int mine = each + (x < rest), before = x * each + min(x, rest);
  if (j < mine) return {true, before + j};
  return {false, x * (a.wgs / 8) - before + j - mine};
}

// Prefix sums of the rows' own tiles into cum[0 .. B), their lengths into ctx; returns
// the total.
template <int KEYS>
__device__ __forceinline__ int scan_own(const SharedArgs& a, int* cum, int* ctx, int* part) {
  const int wave = uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int per = (a.B + 64 * kSplitWaves - 1) / (64 * kSplitWaves), b0 = (int)threadIdx.x * per;
  int sum = 0;
  for (int i = 0; i < per; ++i) {
    const int c = clamped_ctx(a, min(b0 + i, a.B - 1));
    if (b0 + i < a.B) {
      sum += (c - (c < a.P ? 0 : a.P) + KEYS - 1) / KEYS;
      cum[b0 + i] = sum;
      ctx[b0 + i] = c;
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
  int base = incl - sum, total = 0;
#pragma unroll
  for (int w = 0; w < kSplitWaves; ++w) {
    if (w < wave) base += part[w];
    total += part[w];
  }
  for (int i = 0; i < per; ++i)
    if (b0 + i < a.B) {
      const int v = cum[b0 + i] + base;
      cum[b0 + i] = v;
      if (blockIdx.x == 0) a.ws_cum[b0 + i] = v;  // for the joining launch
    }
  __syncthreads();
  return uniform(total);
}

// Where tile u of the rows' own lies.
struct OwnTile {
  int b, vh, tile, tiles;  // row, virtual head, tile of its run, the run's tiles
};
__device__ __forceinline__ OwnTile find_own(const SharedArgs& a, const int* cum, int u) {
  int b = 0;
  for (int hi = a.B - 1; b < hi;) {  // the first row with cum[b] * vheads > u
    const int mid = (b + hi) >> 1;
    if (cum[mid] * a.vheads > u) hi = mid;
    else b = mid + 1;
  }
  const int before = b ? cum[b - 1] : 0, tiles = cum[b] - before, rem = u - before * a.vheads, vh = rem / tiles;
  return {b, vh, rem - vh * tiles, tiles};
}

template <typename T, int DP>
__device__ __forceinline__ void store_own(const SharedArgs& a, const State<DP, 1>& st, int wave_index, int b, int vh,
                                          bool begins) {
  const int lane = (int)threadIdx.x & 63, kvh = vh / a.gsets, g = (vh - kvh * a.gsets) * 16 + (lane & 15);
  const float l = coded_sum(across_groups_sum(st.l[0]), st.any);
  const int64_t slot = begins ? a.own_slot + (int64_t)b * a.Hq + kvh * a.G + g
                              : a.own_cont + (int64_t)wave_index * 16 + (lane & 15);
  if (g < a.G) store_partial<T>(a, st, 0, slot, st.m[0] == kNegInf ? kNegInf : st.mc[0], l);
}
template <typename T, int DP, bool FULL>
__device__ __forceinline__ void load_own_queries(const SharedArgs& a, int b, int vh, uint4 (&qf)[1][Tile<T, DP>::kKS]) {
  const int kvh = vh / a.gsets;
  load_queries<T, DP, 1, FULL>(a, kvh, b * a.G + (vh - kvh * a.gsets) * 16, (b + 1) * a.G, qf);
}

// A wavefront's segment of the rows' own tiles, as one stream over rows and heads:
// the window's lanes find their own tiles, so a run's end costs no new chain of
// loads (length, table, queries, keys), only its partial (24 x 12 heads of 64, f32:
// 23.8 us with a loop over runs, 21.4 so, then 18.3 with all loads unconditional).
template <typename T, int DP, bool FULL, bool NT>
__device__ __forceinline__ void attend_own(const SharedArgs& a, int wave_index, int seg, int total, const int* cum,
                                           const int* ctx) {
  using L = Tile<T, DP>;
  constexpr int kSpan = 64 / L::kGroups;
  const int lane = (int)threadIdx.x & 63;
  if ((int64_t)wave_index * seg >= total) return;
  const int u0 = wave_index * seg, n = min(total - u0, seg);
  const char* kp = (const char*)a.k;
  const char* vp = (const char*)a.v;
  Window win{};
  int row = 0, head = 0;  // of the lane's tile; head: 2 x virtual head, + 1 where the tile begins its run
  auto fill = [&](int t) {
    const int u = u0 + t + lane / L::kGroups;
    if (u < u0 + n) {
      const OwnTile o = find_own(a, cum, u);
      const int c = ctx[o.b], tok = (c < a.P ? 0 : a.P) + o.tile * L::kKeys + 16 * (lane % L::kGroups);
      win = make_window<T>(a, entry_block(a, window_entry(a, o.b, tok), tok), tok, c, o.vh / a.gsets);
      row = o.b;
      head = 2 * o.vh + (o.tile == 0);
    }
  };
  fill(0);
  int b = __builtin_amdgcn_readlane(row, 0), h = __builtin_amdgcn_readlane(head, 0);
  uint4 qf[1][L::kKS];
  State<DP, 1> st;
  L f;
  f32x4 s[1][L::kGroups];
  load_own_queries<T, DP, FULL>(a, b, h >> 1, qf);
  __builtin_amdgcn_sched_barrier(0);
  load_keys<T, DP, FULL, NT>(a, kp, win, 0, f);
  __builtin_amdgcn_sched_barrier(0);
  load_values<T, DP, FULL, NT>(a, vp, win, 0, f);
  __builtin_amdgcn_sched_barrier(0);
  sign_queries(a, qf);
  st.reset();
  for (int t = 0; t + 1 < n; ++t) {  // as in stream_tiles
    const int at = (t + 1) % kSpan * L::kGroups;
    score_tile<T, DP, 1>(f, qf, s);
    if (at == 0) fill(t + 1);
    const int nb = __builtin_amdgcn_readlane(row, at), nh = __builtin_amdgcn_readlane(head, at);
    load_keys<T, DP, FULL, NT>(a, kp, win, at, f);
    const bool ends = nb != b || (nh >> 1) != (h >> 1);
    if (ends) load_own_queries<T, DP, FULL>(a, nb, nh >> 1, qf);
    attend_tile<T, DP, 1, true>(a, f, s, st);
    load_values<T, DP, FULL, NT>(a, vp, win, at, f);
    if (ends) {
      store_own<T>(a, st, wave_index, b, h >> 1, h & 1);
      sign_queries(a, qf);
      st.reset();
      b = nb;
      h = nh;
    }
  }
  score_tile<T, DP, 1>(f, qf, s);
  attend_tile<T, DP, 1, true>(a, f, s, st);
  store_own<T>(a, st, wave_index, b, h >> 1, h & 1);
}

// Own keys and values are read once a call: past what the 256 MB memory-side cache
// may still hold of them they are loaded as non-temporal (64 x 32 heads, 582 MB of
// own tokens: 133 us without, 115 with; 64 x 1, 50 MB, called again and again: 31.5
// and 34.3).
template <typename T, int DP, bool FULL>
__device__ __forceinline__ void attend_own(const SharedArgs& a, int wave_index, int seg, int total, const int* cum,
                                           const int* ctx) {
  if ((int64_t)total * Tile<T, DP>::kKeys * 2 * a.D * (int)sizeof(T) > (int64_t)192 << 20)
    attend_own<T, DP, FULL, true>(a, wave_index, seg, total, cum, ctx);
  else
    attend_own<T, DP, FULL, false>(a, wave_index, seg, total, cum, ctx);
}

// The same for any S, a run at a time.
template <typename T, int DP>
__device__ __forceinline__ void attend_own_any(const SharedArgs& a, int wave_index, int seg, int total, const int* cum,
                                               const int* ctx) {
  using L = Tile<T, DP>;
  if ((int64_t)wave_index * seg >= total) return;
  const int stop = min(total, wave_index * seg + seg);
  uint4 qf[1][L::kKS];
  State<DP, 1> st;
  for (int u = wave_index * seg, n; u < stop; u += n) {
    const OwnTile o = find_own(a, cum, u);
    const int b = uniform(o.b), vh = uniform(o.vh), tile = uniform(o.tile), c = uniform(ctx[b]);
    n = min(uniform(o.tiles) - tile, stop - u);
    load_own_queries<T, DP, false>(a, b, vh, qf);
    st.reset();
    const int first = (c < a.P ? 0 : a.P) + tile * L::kKeys;
    stream_tiles<T, DP, 1, false, false>(
        a, b, vh / a.gsets, first, L::kKeys, [&] { return min(c, first + n * L::kKeys); }, qf, st);
    store_own<T>(a, st, wave_index, b, vh, tile == 0);
  }
}

// The slot of query row r (of a shared piece that begins its run or continues it), or
// -1 where the row takes no part.
__device__ __forceinline__ int64_t shared_slot(const SharedArgs& a, int kvh, int r, int r0, bool begins, int wg) {
  const int rr = min(r, a.B * a.G - 1), b = fast_div(rr, a.g_mul, a.g_shift, a.G), g = rr - b * a.G;
  const int64_t slot = begins ? (int64_t)b * a.Hq + kvh * a.G + g : a.s_cont + (int64_t)wg * a.set_rows + (rr - r0);
  return clamped_ctx(a, b) >= a.P && r == rr ? slot : -1;
}

// Shared pieces from registers, for up to 32 query rows a set and for what the tiles
// in LDS do not take: the workgroup's wavefronts take every fourth tile of a piece
// (a tile of the list is four of theirs) and join in LDS.
template <typename T, int DP, int NQ, bool UNI, bool FULL>
__device__ __forceinline__ void attend_shared(const SharedArgs& a, int wg, int seg,
                                              JoinSpace<DP, NQ, kSplitWaves>& space) {
  using L = Tile<T, DP>;
  const int wave = uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int total = a.s_units * a.s_tiles, step = kSplitWaves * L::kKeys;
  const int team = wg / a.team, member = wg - team * a.team;
  if ((int64_t)team * seg >= total) return;
  const int stop = min(total, team * seg + seg);
  uint4 qf[NQ][L::kKS];
  State<DP, NQ> st;
  for (int u = team * seg, n; u < stop; u += n) {
    const int unit = u / a.s_tiles, tile = u - unit * a.s_tiles, kvh = unit / a.set_blocks;
    const int r0 = ((unit - kvh * a.set_blocks) * a.team + member) * 16 * NQ;
    n = min(a.s_tiles - tile, stop - u);
    if (r0 >= a.B * a.G) continue;
    load_queries<T, DP, NQ, FULL>(a, kvh, r0, a.B * a.G, qf);
    const int64_t slot = shared_slot(a, kvh, r0 + lane % (16 * NQ), r0, tile == 0, wg);
    st.reset();
    stream_tiles<T, DP, NQ, UNI, FULL>(
        a, 0, kvh, tile * step + wave * L::kKeys, step, [&] { return min(a.P, (tile + n) * step); }, qf, st);
    __syncthreads();  // the joins before are done with the space
    if ((int)threadIdx.x < 16 * NQ) space.slot[threadIdx.x] = slot;
    join_waves<T>(a, st, wave, 16 * NQ, space, [&](int row, int d, f32x4 o, float m, float l) {
      const int64_t slot = space.slot[row];
      if (slot < 0) return;
      *(f32x4*)(a.ws_acc + slot * a.D + d) = o;
      if (d == 0) a.ws_ml[slot] = make_float2(m, l);
    });
  }
}

template <typename T, int DP, int NQ, bool UNI, bool FULL>
__global__ void __launch_bounds__(64 * kSplitWaves, DP > 128 ? 1 : 2) paged_shared_split(const SharedArgs a) {
  using Space = JoinSpace<DP, NQ, kSplitWaves>;
  __shared__ __align__(16) char lds[sizeof(Space) > kSharedMaxB * 8 ? sizeof(Space) : kSharedMaxB * 8];
  __shared__ int part[kSplitWaves];
  int *cum = (int*)lds, *ctx = cum + kSharedMaxB;
  const int total = scan_own<Tile<T, DP>::kKeys>(a, cum, ctx, part) * a.vheads;
  const Split sp = make_split(a, total);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.ws_split[0] = sp.seg_shared, a.ws_split[1] = sp.seg_own;
  const Place at = make_place(a, sp);
  if (at.shared) {
    attend_shared<T, DP, NQ, UNI, FULL>(a, at.index, sp.seg_shared, *(Space*)lds);
  } else {
    const int w = at.index * kSplitWaves + uniform((int)threadIdx.x >> 6);
    if constexpr (UNI) attend_own<T, DP, FULL>(a, w, sp.seg_own, total, cum, ctx);
    else attend_own_any<T, DP>(a, w, sp.seg_own, total, cum, ctx);
  }
}

// ------------------------------------------------- shared tiles in LDS
// For more query rows than registers hold: the workgroup's four wavefronts hold 16 QB
// rows each and read the same 64-key tiles from LDS, copied there straight from
// memory one tile ahead, so a key is read from L2 once per 64 QB rows (128 x 32 heads
// on 8 KV heads over 65 536 tokens: 360 us from registers with 64 rows to a
// wavefront, 204 through LDS). Each wavefront copies 16 of a tile's rows: one group
// of the block table's, at a scalar base. As in paged_prefill_tr, S^T's rows are the
// keys 32 c + 8 (r / 4) + 4 h + r % 4 for block 2 c + h, which puts 8 consecutive keys
// of its column into a lane, and V^T comes out of ds_read_b64_tr_b16; the weights'
// sums are one more product, with ones. s_setprio puts a wavefront's products before
// the other's softmax on its SIMD (156 -> 149 us without own tokens).
template <typename T, int DP, int QB>
struct LdsState {
  f32x4 acc[QB][DP / 16], sum[QB];
  float m[QB], mc[QB];
};

template <typename T, int DP, int QB>
__device__ __forceinline__ void attend_lds_tile(const SharedArgs& a, const char* kl, uint32_t vl, uint32_t counts,
                                                const uint4 (&qf)[QB][DP / 32], LdsState<T, DP, QB>& st) {
  constexpr int kRowB = DP * 2, kCPR = DP / 8;
  const int lane = (int)threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int kr = 8 * (col >> 2) + (col & 3);
  f32x4 s[QB][4];
  // The next block's keys are read before this one's products; left to itself the
  // compiler waits for every read.
  uint4 kv[2][DP / 32];
  auto read = [&](int kb) {
#pragma unroll
    for (int f = 0; f < DP / 32; ++f)
      kv[kb & 1][f] = *(const uint4*)(kl + (kr + 32 * (kb >> 1) + 4 * (kb & 1)) * kRowB +
                                      (((4 * f + g) ^ k_swz<kCPR>(kr)) << 4));
  };
  read(0);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
    if (kb < 3) read(kb + 1);
#pragma unroll
    for (int q = 0; q < QB; ++q) s[q][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < DP / 32; ++f)
#pragma unroll
      for (int q = 0; q < QB; ++q) s[q][kb] = mfma16<T>(kv[kb & 1][f], qf[q][f], s[q][kb]);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
  // The first half of V^T is read under the softmax, the second as the first's products
  // let go of its registers.
  const int vrow = 8 * g + (col >> 2), vq = lane & 3;
  uint4 vv[DP / 16];
  auto value = [&](int h, int t) {
    const uint32_t at = vl + (vrow + 32 * h) * kRowB + ((vq & 1) << 3) +
                        (((2 * t + (vq >> 1)) ^ v_swz<kCPR>(vrow)) << 4);
    const uint2 lo = TrRead<T>::at(at), hi = TrRead<T>::at(at + 4 * kRowB);
    vv[t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
#pragma unroll
  for (int t = 0; t < DP / 16; ++t) value(0, t);
  __builtin_amdgcn_sched_barrier(0);
  if (counts != 0x10101010u) {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const int j = 2 * (kb >> 1) + (g >> 1), first = 8 * (g & 1) + 4 * (kb & 1), n = (int)(counts >> (8 * j)) & 255;
#pragma unroll
      for (int q = 0; q < QB; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[q][kb][i] = first + i < n ? s[q][kb][i] : kNegInf;
    }
  }
  const float c = a.scale_log2;
  uint4 pf[QB][2];
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    float top = kNegInf;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[q][kb][i]);
    if (__any(top > st.m[q] + a.lazy)) {
      const float mn = fmaxf(st.m[q], across_groups_max(top)), mcn = exponent_base<T>(mn, c);
      const float alpha = st.m[q] == kNegInf ? 0.f : fast_exp2(st.mc[q] - mcn);
      st.m[q] = mn;
      st.mc[q] = mcn;
      st.sum[q] *= alpha;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) st.acc[q][t] *= alpha;
    }
    float p[16];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[4 * kb + i] = fast_exp2(fmaf(s[q][kb][i], c, -st.mc[q]));
#pragma unroll
    for (int h = 0; h < 2; ++h)
      pf[q][h] = make_uint4(pack2<T>(p[8 * h], p[8 * h + 1]), pack2<T>(p[8 * h + 2], p[8 * h + 3]),
                            pack2<T>(p[8 * h + 4], p[8 * h + 5]), pack2<T>(p[8 * h + 6], p[8 * h + 7]));
  }
  const uint32_t one2 = pack2<T>(1.f, 1.f);
  const uint4 ones = make_uint4(one2, one2, one2, one2);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
#pragma unroll
      for (int q = 0; q < QB; ++q) st.acc[q][t] = mfma16<T>(vv[t], pf[q][h], st.acc[q][t]);
      if (h == 0) value(1, t);
    }
#pragma unroll
    for (int q = 0; q < QB; ++q) st.sum[q] = mfma16<T>(ones, pf[q][h], st.sum[q]);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

template <typename T, int DP, int QB>
__device__ __forceinline__ void attend_shared_lds(const SharedArgs& a, int wg, int seg, char* lds) {
  constexpr int kRowB = DP * 2, kCPR = DP / 8, kTileB = 64 * kRowB, kRPC = 1024 / kRowB, kCopies = 16 / kRPC;
  const int wave = uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int total = a.s_units * a.s_tiles;
  const int team = wg / a.team, member = wg - team * a.team;
  if ((int64_t)team * seg >= total) return;
  const int stop = min(total, team * seg + seg);
  // The lane's part of the wavefront's copies: row c * kRPC + lane / kCPR of its 16, and
  // the chunk of it that the swizzles place there.
  auto copy_row = [&](int c, int l) { return c * kRPC + l / kCPR; };
  auto k_chunk = [&](int c, int l) { return (l % kCPR) ^ k_swz<kCPR>(16 * wave + copy_row(c, l)); };
  auto v_chunk = [&](int c, int l) { return (l % kCPR) ^ v_swz<kCPR>(16 * wave + copy_row(c, l)); };
  uint32_t ko[kCopies], vo[kCopies];
#pragma unroll
  for (int c = 0; c < kCopies; ++c) {
    ko[c] = (uint32_t)copy_row(c, lane) * (uint32_t)a.k_ss * 2 + (uint32_t)k_chunk(c, lane) * 16;
    vo[c] = (uint32_t)copy_row(c, lane) * (uint32_t)a.v_ss * 2 + (uint32_t)v_chunk(c, lane) * 16;
  }
  const uint32_t dst0 = lds_addr(lds) + (uint32_t)wave * 16 * kRowB;
  const bool all_dims = a.D == DP;
  uint4 qf[QB][DP / 32];
  LdsState<T, DP, QB> st;
  for (int u = team * seg, n; u < stop; u += n) {
    const int unit = u / a.s_tiles, tile0 = u - unit * a.s_tiles, kvh = unit / a.set_blocks;
    const int r0 = ((unit - kvh * a.set_blocks) * a.team + member) * 64 * QB, mine = r0 + wave * 16 * QB;
    n = min(a.s_tiles - tile0, stop - u);
    if (r0 >= a.B * a.G) continue;  // the last block's teams may be short
    // A window of 64 tiles: lane i holds tile i's four groups' key counts and the
    // place of the wavefront's own.
    Window win{};
    uint32_t counts = 0;
    uint32_t now = 0, next = 0;  // key counts of the tile computed and of the one copied
    auto copy = [&](int i, int stage) {
      if (i % 64 == 0) {
        const int tok = (tile0 + i + lane) * 64;
        Index entry[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) entry[j] = window_entry(a, 0, tok + 16 * j);
        counts = 0;
        int id_own = -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int id = entry_block(a, entry[j], tok + 16 * j);
          counts |= (uint32_t)(id < 0 ? 0 : max(0, min(16, a.P - tok - 16 * j))) << (8 * j);
          if (wave == j) id_own = id;
        }
        win = make_window<T>(a, id_own, tok + 16 * wave, a.P, kvh);
      }
      const int at = i % 64;
      next = (uint32_t)__builtin_amdgcn_readlane((int)counts, at);
      const char* kb = (const char*)a.k + lane_offset(win.k_lo, win.k_hi, at);
      const char* vb = (const char*)a.v + lane_offset(win.v_lo, win.v_hi, at);
      uint32_t kd = dst0 + stage * 2 * kTileB, vd = kd + kTileB;
      if (all_dims && next == 0x10101010u) {
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          copy16_to_lds(kb, ko[c], kd + 1024 * c);
          copy16_to_lds(vb, vo[c], vd + 1024 * c);
        }
      } else {  // what does not count is zeros
        const int m = (int)(next >> (8 * wave)) & 255;
        int l = lane;
        asm volatile("" : "+v"(l));  // keeps this rare path's rows and chunks out of the loop's registers
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          const int kc = k_chunk(c, l), vc = v_chunk(c, l);
          const bool ok = copy_row(c, l) < m;
          const char* zero = (const char*)kZeroRow;
          const char* ks = ok && kc * 8 < a.D ? kb + ko[c] : zero + kc * 16;
          const char* vs = ok && vc * 8 < a.D ? vb + vo[c] : zero + vc * 16;
          copy16_to_lds(ks, kd + 1024 * c);
          copy16_to_lds(vs, vd + 1024 * c);
        }
      }
    };
    load_queries<T, DP, QB, false>(a, kvh, mine, a.B * a.G, qf);
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      st.sum[q] = f32x4{0.f, 0.f, 0.f, 0.f};
      st.m[q] = kNegInf;
      st.mc[q] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) st.acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool any = false;
    const bool active = mine < a.B * a.G;
    __syncthreads();  // the tiles of the piece before, and the scan's sums, are done with
    copy(0, 0);
    sign_queries(a, qf);
    auto turn = [&](int i, auto stage) {
      constexpr int S = decltype(stage)::value;
      now = next;
      wait_and_barrier<0>();  // tile i has landed, and tile i - 1 is done with
      if (i + 1 < n) copy(i + 1, S ^ 1);
      any |= now != 0;
      if (active)
        attend_lds_tile<T, DP, QB>(a, lds + S * 2 * kTileB, lds_addr(lds) + S * 2 * kTileB + kTileB, now, qf, st);
    };
    for (int i = 0; i < n; i += 2) {
      turn(i, Stage<0>{});
      if (i + 1 < n) turn(i + 1, Stage<1>{});
    }
    int64_t slots[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q) slots[q] = shared_slot(a, kvh, mine + 16 * q + col, r0, tile0 == 0, wg);
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      const int64_t slot = slots[q];
      if (slot < 0) continue;
      if (lane < 16)
        a.ws_ml[slot] = make_float2(st.m[q] == kNegInf ? kNegInf : st.mc[q], coded_sum(st.sum[q][0], any));
      float* out = a.ws_acc + slot * a.D + 4 * g;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t)
        if (16 * t + 4 * g < a.D) *(f32x4*)(out + 16 * t) = st.acc[q][t];
    }
  }
}

template <typename T, int DP, int QB, bool FULL>
__global__ void __launch_bounds__(64 * kSplitWaves, 2) paged_shared_split_lds(const SharedArgs a) {
  __shared__ __align__(1024) char lds[4 * 64 * DP * 2];
  __shared__ int part[kSplitWaves];
  static_assert(sizeof(lds) >= kSharedMaxB * 8, "the rows' prefix sums and lengths fit the tiles' place");
  int *cum = (int*)lds, *ctx = cum + kSharedMaxB;
  const int total = scan_own<Tile<T, DP>::kKeys>(a, cum, ctx, part) * a.vheads;
  const Split sp = make_split(a, total);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.ws_split[0] = sp.seg_shared, a.ws_split[1] = sp.seg_own;
  const Place at = make_place(a, sp);
  if (at.shared) {
    attend_shared_lds<T, DP, QB>(a, at.index, sp.seg_shared, lds);
  } else {
    attend_own<T, DP, FULL>(a, at.index * kSplitWaves + uniform((int)threadIdx.x >> 6), sp.seg_own, total, cum, ctx);
  }
}

// Joins the partials of one (row, query head) per JW wavefronts: lanes over the
// pieces for their weights, then D / 4 lanes to a piece's row.
template <typename T, int JW>
__global__ void __launch_bounds__(256) paged_shared_join(const SharedArgs a) {
  __shared__ f32x4 part[4][64];
  __shared__ float ml[4][2];
  const int wave = uniform((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (4 / JW) + wave / JW;
  const bool live = unit < (int64_t)a.B * a.Hq;
  const int b = live ? (int)(unit / a.Hq) : 0, hq = live ? (int)(unit - (int64_t)b * a.Hq) : 0;
  const int kvh = hq / a.G, g = hq - kvh * a.G, set = g / 16, r = b * a.G + g;
  const int last = a.ws_cum[max(b - 1, 0)], upto = a.ws_cum[b], seg_shared = a.ws_split[0], seg_own = a.ws_split[1];
  const int ctx = clamped_ctx(a, b), before = b ? last : 0, tiles = upto - before;
  int shared = 0, s0 = 0, member = 0, pieces = 0, w0 = 0;
  if (a.s_tiles && ctx >= a.P) {
    const int rs = r / a.set_rows, u = (kvh * a.set_blocks + rs / a.team) * a.s_tiles;
    member = rs % a.team;
    s0 = u / seg_shared;
    shared = (u + a.s_tiles - 1) / seg_shared - s0 + 1;
  }
  if (tiles) {
    const int u = before * a.vheads + (kvh * a.gsets + set) * tiles;
    w0 = u / seg_own;
    pieces = (u + tiles - 1) / seg_own - w0 + 1;
  }
  const int n = live ? shared + pieces : 0;
  auto slot = [&](int i) -> int64_t {
    if (i < shared)
      return i == 0 ? unit : a.s_cont + ((int64_t)(s0 + i) * a.team + member) * a.set_rows + r % a.set_rows;
    i -= shared;
    return i == 0 ? a.own_slot + unit : a.own_cont + (int64_t)(w0 + i) * 16 + (g - set * 16);
  };
  const int lpr = a.D <= 64 ? 16 : a.D <= 128 ? 32 : 64, at = lane / lpr, d = 4 * (lane % lpr), per = 64 / lpr;
  constexpr int kEarly = 8;
  float top = kNegInf, sum = 0.f;
  bool dead = false;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int share = (n + JW - 1) / JW, stop = min(n, (wave % JW + 1) * share);  // the wavefront's pieces
  for (int i0 = wave % JW * share; i0 < stop; i0 += 64) {
    const int m = min(64, stop - i0);
    // The first pieces' rows load beside the weights that say whether they count (64 x 8
    // heads, some 20 pieces each: 6.6 us after them, 5.5 so; 128 x 32: 11.2 and 9.8).
    f32x4 early[kEarly];
#pragma unroll
    for (int j = 0; j < kEarly; ++j) {
      const int i = j * per + at;
      early[j] = i < m && d < a.D ? *(const f32x4*)(a.ws_acc + slot(i0 + i) * a.D + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float2 x = lane < m ? a.ws_ml[slot(i0 + lane)] : make_float2(kNegInf, 0.f);
    const bool counts = !(x.y <= 0.f);
    dead |= x.y < 0.f;
    const float mn = fmaxf(top, wave_max(counts ? x.x : kNegInf));
    const float alpha = top == kNegInf ? 0.f : fast_exp2(top - mn);
    const float w = counts ? fast_exp2(x.x - mn) : 0.f;
    sum = sum * alpha + wave_sum(counts ? x.y * w : 0.f);
    acc *= alpha;
    top = mn;
    // Every lane takes part in the exchanges: a lane reads one that is switched off as 0.
#pragma unroll
    for (int j = 0; j < kEarly; ++j) {
      if (j * per >= m) break;
      const float wi = __shfl(w, j * per + at, 64);
      const int use = __shfl((int)counts, j * per + at, 64);
      if (use && j * per + at < m) acc += wi * early[j];
    }
#pragma unroll 8
    for (int i = kEarly * per; i < m; i += per) {
      const float wi = __shfl(w, i + at, 64);
      const int use = __shfl((int)counts, i + at, 64);
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (use && i + at < m && d < a.D) v = *(const f32x4*)(a.ws_acc + slot(i0 + i + at) * a.D + d);
      acc += wi * v;
    }
  }
#pragma unroll
  for (int m = 32; m >= 16; m >>= 1)
    if (lpr <= m) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], m, 64);
    }
  dead = __any(dead);
  if constexpr (JW > 1) {
    if (lane == 0) ml[wave][0] = top, ml[wave][1] = sum == 0.f && dead ? -1.f : sum;
    part[wave][lane] = acc;
    __syncthreads();
    if (wave % JW) return;
    float tn = kNegInf, sn = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    dead = false;
#pragma unroll
    for (int w = 0; w < JW; ++w)
      if (!(ml[wave + w][1] <= 0.f)) tn = fmaxf(tn, ml[wave + w][0]);
#pragma unroll
    for (int w = 0; w < JW; ++w) {
      const float l = ml[wave + w][1];
      dead |= l < 0.f;
      if (l <= 0.f) continue;
      const float f = fast_exp2(ml[wave + w][0] - tn);
      sn += l * f;
      acc += f * part[wave + w][lane];
    }
    sum = sn;
  }
  const float inv = sum == 0.f ? (dead ? __builtin_nanf("") : 0.f) : 1.f / sum;
  if (live && at == 0 && d < a.D) {
    T* o = (T*)a.out + (int64_t)b * a.o_sb + (int64_t)hq * a.o_sh + d;
    if constexpr (sizeof(T) == 4) *(f32x4*)o = acc * inv;
    else *(uint2*)o = make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
  }
}

// One workgroup per (row, virtual head): all of the row's tokens in one launch.
template <int DP>
constexpr int kOneWaves = DP > 128 ? 4 : 8;
template <typename T, int DP, bool UNI, bool FULL>
__global__ void __launch_bounds__(64 * kOneWaves<DP>) paged_shared_one(const SharedArgs a) {
  using L = Tile<T, DP>;
  __shared__ __align__(16) JoinSpace<DP, 1, kOneWaves<DP>> space;
  const int wave = uniform((int)threadIdx.x >> 6);
  const int b = (int)blockIdx.y, vh = (int)blockIdx.x, kvh = vh / a.gsets, g0 = (vh - kvh * a.gsets) * 16;
  uint4 qf[1][L::kKS];
  State<DP, 1> st;
  load_queries<T, DP, 1, FULL>(a, kvh, b * a.G + g0, (b + 1) * a.G, qf);
  const Index ctx = ctx_load(a, b);
  st.reset();
  stream_tiles<T, DP, 1, UNI, FULL>(
      a, b, kvh, wave * L::kKeys, kOneWaves<DP> * L::kKeys, [&] { return ctx_value(a, ctx); }, qf, st);
  join_waves<T>(a, st, wave, min(16, a.G - g0), space, [&](int row, int d, f32x4 o, float, float l) {
    const f32x4 x = o * (l == 0.f ? 0.f : l < 0.f ? __builtin_nanf("") : 1.f / l);
    T* p = (T*)a.out + (int64_t)b * a.o_sb + (int64_t)(kvh * a.G + g0 + row) * a.o_sh + d;
    if constexpr (sizeof(T) == 4) *(f32x4*)p = x;
    else *(uint2*)p = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
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
  if constexpr (DP <= 128)
    if (a.row_tiles == 2) fn = (const void*)&paged_shared_split<T, DP, 2, UNI, FULL>;
  if constexpr (sizeof(T) == 2 && DP <= 128 && UNI) {
    if (a.lds_tiles)
      fn = a.row_tiles == 2 ? (const void*)&paged_shared_split_lds<T, DP, 2, FULL>
                            : (const void*)&paged_shared_split_lds<T, DP, 1, FULL>;
  }
  const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)a.wgs), dim3(64 * kSplitWaves), kargs, 0, stream);
  if (e != hipSuccess) return e;
  // Four wavefronts join a row's pieces where there are many: at most so many of either kind.
  const int64_t units = (int64_t)a.B * a.Hq;
  const int64_t most = 2 + (int64_t)a.wgs * kSplitWaves / ((int64_t)a.B * a.vheads) +
                       (a.s_units ? a.wgs / (a.s_units * a.team) : 0);
  if (most > 24)
    return hipLaunchKernel((const void*)&paged_shared_join<T, 4>, dim3((unsigned)units), dim3(256), kargs, 0, stream);
  return hipLaunchKernel((const void*)&paged_shared_join<T, 1>, dim3((unsigned)((units + 3) / 4)), dim3(256), kargs, 0,
                         stream);
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
    return hipLaunchKernel((const void*)&paged_shared_any<T>, dim3((unsigned)a.Hq, (unsigned)a.B), dim3(64), kargs, 0,
                           stream);
  }
  return a.D <= 64    ? launch_width<T, 64>(a, stream)
         : a.D <= 128 ? launch_width<T, 128>(a, stream)
                      : launch_width<T, 256>(a, stream);
}

}  // namespace

}  // namespace mgi
