// prompt_attention.h -- causal attention of whole prompts, packed one after the other, on
// the matrix cores of gfx950. Keys and values are the projection's own rows (no pool);
// query heads may share KV heads.
//
//   out[i,h] = sum_{j <= i} softmax_j(scale * q[i,h] . k[j, h / G]) v[j, h / G]
// over the rows j of i's sequence. 4 D flops per (query head, visible pair of rows), and
// each K and V row is used by every later row: bound by the matrix cores and by the
// exponentials beside them (per score 2 D / 512 matrix cycles of a SIMD, 16 for the
// exponential, about 10 for the rest), from a few hundred tokens on.
//
// A workgroup is four wavefronts of 32 query rows each: the same 32 positions of four heads
// that share a KV head, 64 positions of two, or 128 of one. Keys and values stream
// through LDS in tiles, two in flight, copied there straight from memory. Each wavefront
// computes S^T = K Q^T and O^T += V^T P^T with 32x32 MFMAs, so a lane's column is one
// query row: its running maximum and sum are the lane's own (two lanes share a row), and
// S^T's rows (keys 8 (r / 4) + 4 (lane / 32) + r % 4) are the order in which P^T enters the
// second product when V^T's keys are read in the same order.
//
// Work order: the work of a tile of positions grows with its index in its sequence, so
// workgroups take all sequences' tiles in falling index, which every workgroup finds from
// the sequence starts by itself: nothing is read on the host, and no launch precedes it.
//
// Measured on MI355X: three prompts of 4000-8192 tokens, 32 heads of 128 on 8, bf16, 1020 us
// (1.08 PFLOP/s; the library's 8192^3 product reaches 1.36); 24 of 20-1500 169 us; f16, 7 of
// 300-2100, 20 heads of 80, 76 us. In the first the matrix cores are busy 48 % of all cycles, at
// 1.9 GHz; a 64-key tile takes 2760 cycles of two wavefronts to a SIMD (2210 if nothing were
// waited for), and a workgroup 18k more for its search, first copies, diagonal and output,
// which is what bounds short prompts.
//
// Numerics: f32 sums and softmax (log2 domain). 2-byte types round the weights to their
// type for the second product, half a step each (bf16 2^-8 of a weight at most, f16 2^-11; the
// errors are independent), and the sum that divides is that of the rounded weights; f16 weights are scaled by 2^13, so that
// far keys keep theirs. f32 multiplies in f32. The maximum is taken from the scores themselves where
// they are large, not from their rounded products with the scale: any finite score gives a
// finite weight (one more test per 32 keys: 0.6-1.1 % of the calls above).
#pragma once

#include <algorithm>
#include <type_traits>

#include "lds_tiles.h"
#include "mgi_common.h"
#include "minivllm_hip.h"
#include "prompt_args.h"

namespace mgi {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <typename T> struct PM;  // the products of a type
template <> struct PM<bf16_t> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  // log2: a score may pass the maximum by slack; weights are 2^bias too large, so that no sum is larger than the softmax's.
  static constexpr float slack = 8.f, bias = -8.f;
  static constexpr uint32_t inf = 0x7f80u;  // bits
  __device__ static __forceinline__ f32x16_t mfma(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack2(float lo, float hi) {
    const f32x2_t x = {lo, hi};  // converted as a vector: one instruction (three, element by element)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, v2));
  }
  __device__ static __forceinline__ float sum2(uint32_t w, float acc) {
    const v2 one = {(__bf16)1.f, (__bf16)1.f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w), one, acc, false);
  }
};
template <> struct PM<f16_t> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static constexpr float slack = 2.f, bias = 13.f;  // f16 values leave f32 sums the room
  static constexpr uint32_t inf = 0x7c00u;
  __device__ static __forceinline__ f32x16_t mfma(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack2(float lo, float hi) {
    const v2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
  __device__ static __forceinline__ float sum2(uint32_t w, float acc) {
    const v2 one = {(_Float16)1.f, (_Float16)1.f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, w), one, acc, false);
  }
};
template <> struct PM<float> {
  static constexpr float slack = 8.f, bias = -8.f;
};

template <typename T> struct PElem {
  __device__ static __forceinline__ uint32_t bits(const T* p) { return p->bits; }
};
template <> struct PElem<float> {
  __device__ static __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
};

// Sum and maximum over the wavefront of numbers that are not negative, by DPP.
template <typename Op>
__device__ __forceinline__ int wave_reduce(int x, Op op) {
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));  // lanes 1, 2, 4 and 8 below in the row
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true));  // row 0's last to row 1, 2's to 3
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true));  // row 1's last to rows 2 and 3
  return __builtin_amdgcn_readlane(x, 63);
}

__device__ __forceinline__ float uniform(float x) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}

struct Span {
  int start, rows;
};
__device__ __forceinline__ int64_t clamped(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }
__device__ __forceinline__ Span span_of(const PromptArgs& a, int b) {
  Index s, e;  // both loads before either's use
  s.load(a.starts, a.cu_i64, (uint64_t)min(b, a.B) * (uint64_t)a.cu_s);
  e.load(a.starts, a.cu_i64, (uint64_t)min(b + 1, a.B) * (uint64_t)a.cu_s);
  const int lo = (int)clamped(s.value(a.cu_i64), 0, a.T), hi = (int)clamped(e.value(a.cu_i64), lo, a.T);
  return Span{lo, hi - lo};
}

// The `rank`-th tile (of `rows` positions) in falling order of its index in its sequence:
// the sequence's rows and the index, or no rows past the last. The first kKept sequences'
// lengths stay in registers, the others' are read again in each step of the search.
struct PromptTile {
  Span seq;
  int index;
};
__device__ __forceinline__ PromptTile tile_at(const PromptArgs& a, int rank, int rows) {
  constexpr int kKept = 4;
  const int lane = (int)(threadIdx.x & 63), shift = __builtin_ctz(rows);
  const auto tiles = [&](Span x) { return (x.rows + rows - 1) >> shift; };
  Span kept[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) kept[i] = 64 * i < a.B ? span_of(a, 64 * i + lane) : Span{0, 0};
  const auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kKept; ++i)
      if (64 * i < a.B) f(kept[i]);
    for (int b0 = 64 * kKept; b0 < a.B; b0 += 64) f(span_of(a, b0 + lane));
  };
  const auto sum = [](int x, int y) { return x + y; };
  const auto larger = [](int x, int y) { return max(x, y); };
  int most = 0;
  each([&](Span x) { most = max(most, tiles(x)); });
  most = wave_reduce(most, larger);
  const auto from = [&](int index) __attribute__((always_inline)) {  // tiles with this index or a higher one
    int n = 0;
    each([&](Span x) { n += max(0, tiles(x) - index); });
    return wave_reduce(n, sum);
  };
  if (rank >= from(0)) return PromptTile{Span{0, 0}, 0};
  int lo = 0, hi = most, above = 0;  // from(lo) > rank >= from(hi) = above
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, n = from(mid);
    if (n > rank) lo = mid;
    else hi = mid, above = n;
  }
  int left = rank - above;
  PromptTile found{Span{0, 0}, lo};
  each([&](Span x) {
    if (left < 0) return;
    const bool has = tiles(x) > lo;
    const uint64_t all = __ballot(has);
    const int count = __popcll(all);
    if (left < count) {
      const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
      const int at = __ffsll((unsigned long long)__ballot(has && before == left)) - 1;
      found.seq = Span{__builtin_amdgcn_readlane(x.start, at), __builtin_amdgcn_readlane(x.rows, at)};
    }
    left -= count;
  });
  return found;
}

// DP: head dim, padded to a multiple of 16 (D <= DP). VEC: rows are copied in 16-byte pieces.
template <typename T, int DP, bool VEC>
struct Prompt {
  static constexpr int EB = (int)sizeof(T);
  static constexpr bool F32 = EB == 4;
  static constexpr int NDB = (DP + 31) / 32;        // 32-wide blocks of O^T's dims
  static constexpr int ROWB = NDB * 32 * EB;        // bytes of a row in LDS
  static constexpr int CPR = ROWB / 16;             // 16-byte chunks of a row
  static constexpr int EPC = 16 / EB;               // elements of a chunk
  static constexpr int KT = F32 ? 32 : 64;          // keys of a tile
  static constexpr int TILEB = KT * ROWB;
  static constexpr int COPIES = TILEB / 4096;       // 16-byte copies per lane, tile and tensor
  static_assert(COPIES * 4096 == TILEB, "the workgroup copies whole tiles");
  static constexpr int NF = DP / (2 * EPC);         // steps of the first product: two chunks each
  static constexpr int NKB = KT / 32;
  // Workgroups of a CU, by their LDS (and for unaligned f32 rows by registers: two would spill them).
  static constexpr int RESIDENT = 4 * TILEB > 80 * 1024 || (F32 && !VEC && DP >= 128) ? 1 : 2;
  static constexpr int PREGS = F32 ? 16 : 8;        // registers of a 32-key block's weights
  using M = PM<T>;

  // A chunk's place in its row: spread over the banks that rows would share. K reads take
  // one chunk of 32 rows; V reads 8 (f32: 2) neighbouring rows' chunks of one block of dims.
  // Of LDS cycles, conflicts are 1.5 % for heads of 128 and 256, 2-byte types; where a row is not 16
  // or 32 chunks, its stride separates some of the same row bits already: 33 % for 64 and 192, 60 % for
  // 32, 58 % for 80. f32 heads of 64 and 128: none.
  __device__ static __forceinline__ int k_place(int row, int c) {
    constexpr int bits = CPR % 16 == 0 ? 15 : CPR % 8 == 0 ? 7 : 3;
    return c ^ (row & bits);
  }
  __device__ static __forceinline__ int v_place(int row, int c) {
    if constexpr (F32) return c;
    else return CPR % 16 == 0 ? c ^ (4 * (row & 3)) : CPR % 8 == 0 ? c ^ (4 * ((row >> 1) & 1)) : c;
  }

  // A word of V (f32, or two halves) with 0 for what is not a number or infinite.
  __device__ static __forceinline__ uint32_t finite(uint32_t w) {
    if constexpr (F32) {
      return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
    } else {
      if ((w & 0x7fffu) >= M::inf) w &= 0xffff0000u;
      return ((w >> 16) & 0x7fffu) >= M::inf ? w & 0xffffu : w;
    }
  }

  // Copy i of a whole tile (see copy): from `base`, its first key's row.
  template <bool KEYS, int I>
  __device__ static __forceinline__ void copy_piece(const PromptArgs& a, const char* base, int64_t st, uint32_t dst) {
    const int at = I * 256 + (int)threadIdx.x, row = at / CPR, place = at % CPR;
    const int c = KEYS ? k_place(row, place) : v_place(row, place);  // its own inverse
    const uint32_t off = (uint32_t)row * (uint32_t)(st * EB) + (c * EPC < a.D ? (uint32_t)c * 16 : 0u);
    copy16_to_lds(base, off, __builtin_amdgcn_readfirstlane(dst + (uint32_t)(I * 256 + ((int)threadIdx.x & ~63)) * 16));
  }

  // One tile (keys key0 .. of this sequence) of K or V into LDS at `dst`, by all four wavefronts.
  template <bool KEYS>
  __device__ static __forceinline__ void copy(const PromptArgs& a, const T* head, int64_t st, int64_t sd, int key0, int n,
                                              uint32_t dst, unsigned char* lds) {
    // Chunks past D: of K zeros, which queries padded with zeros need; of V anything, for
    // the dims past D are not written.
    const bool whole = key0 + KT <= n && (!KEYS || a.D == DP);
    const char* base = (const char*)(head + (int64_t)key0 * st);
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const int at = i * 256 + (int)threadIdx.x, row = at / CPR, place = at % CPR;
        const int c = KEYS ? k_place(row, place) : v_place(row, place);  // its own inverse
        const uint32_t off = (uint32_t)row * (uint32_t)(st * EB) + (c * EPC < a.D ? (uint32_t)c * 16 : 0u);
        const uint32_t to = __builtin_amdgcn_readfirstlane(dst + (uint32_t)(i * 256 + ((int)threadIdx.x & ~63)) * 16);
        if (whole) {
          copy16_to_lds(base, off, to);
        } else {
          const bool in = key0 + row < n && c * EPC < a.D;
          copy16_to_lds(in ? base + off : (const char*)kZeroRow, to);
        }
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < COPIES; ++i) {
        const int at = i * 256 + (int)threadIdx.x, row = at / CPR, place = at % CPR;
        const int c = KEYS ? k_place(row, place) : v_place(row, place);
        uint32_t w[4] = {0, 0, 0, 0};
        if (key0 + row < n) {
          const T* p = (const T*)base + (int64_t)row * st;
#pragma unroll
          for (int e = 0; e < EPC; ++e)
            if (c * EPC + e < a.D) w[e * EB / 4] |= PElem<T>::bits(p + (c * EPC + e) * sd) << (8 * (e * EB % 4));
        }
        *(uint4*)(lds + at * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
};

template <typename T, int DP, bool VEC>
__global__ void __launch_bounds__(256, (Prompt<T, DP, VEC>::RESIDENT))
prompt_attention_kernel(const PromptArgs a) {
  using P = Prompt<T, DP, VEC>;
  using M = PM<T>;
  constexpr int NDB = P::NDB, NF = P::NF, NKB = P::NKB, KT = P::KT, ROWB = P::ROWB, TILEB = P::TILEB;
  __shared__ __align__(1024) unsigned char lds[4][TILEB];  // two tiles of keys, two of values
  unsigned char(*k_lds)[TILEB] = lds;
  unsigned char(*v_lds)[TILEB] = lds + 2;

  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, kg = lane >> 5;

  // Rows of no sequence: before the first start, behind the last.
  if (a.zero_rest) {
    const int64_t s0 = load_index(a.starts, a.cu_i64, 0), s1 = load_index(a.starts, a.cu_i64, (int64_t)a.B * a.cu_s);
    const int lo = (int)(s0 < 0 ? 0 : s0 > a.T ? a.T : s0), hi = (int)(s1 < lo ? lo : s1 > a.T ? a.T : s1);
    const int rest = lo + a.T - hi;
    for (int r = (int)blockIdx.x; r < rest; r += (int)gridDim.x) {
      T* row = (T*)a.out + (int64_t)(r < lo ? r : hi + r - lo) * a.o_st;
      for (int i = tid; i < a.Hq * a.D; i += 256) {
        const int h = i / a.D;
        Elem<T>::store(row + h * a.o_sh + (i - h * a.D) * a.o_sd, 0.f);
      }
    }
  }

  // This workgroup's tile of positions and heads; head groups fastest, so that those of
  // one KV head tend to one XCD.
  const int hgroups = a.Hq / a.heads, rows = kPromptRows / a.heads;
  const int rank = (int)blockIdx.x / hgroups, hg = (int)blockIdx.x - rank * hgroups;
  const PromptTile tile = tile_at(a, rank, rows);
  const int n = tile.seq.rows, start = tile.seq.start;
  if (n == 0) return;
  const int per_head = 4 / a.heads;                    // wavefronts of one head
  const int h = hg * a.heads + wave / per_head, kvh = h / a.G;
  const int first = tile.index * rows + wave % per_head * 32;  // this wavefront's first position
  const int last = min(n, first + 32) - 1;             // below first: the wavefront has no rows
  const int pos = first + col;
  const int end = min(n, (tile.index + 1) * rows);     // positions the workgroup's keys reach
  const int steps = (end + KT - 1) / KT;

  const T* kh = (const T*)a.k + (int64_t)start * a.k_st + (int64_t)kvh * a.k_sh;
  const T* vh = (const T*)a.v + (int64_t)start * a.v_st + (int64_t)kvh * a.v_sh;
  const auto issue_keys = [&](int step, int buf) __attribute__((always_inline)) {
    P::template copy<true>(a, kh, a.k_st, a.k_sd, step * KT, n, lds_addr(k_lds[buf]), k_lds[buf]);
  };
  const auto issue_values = [&](int step, int buf) __attribute__((always_inline)) {
    P::template copy<false>(a, vh, a.v_st, a.v_sd, step * KT, n, lds_addr(v_lds[buf]), v_lds[buf]);
  };

  issue_keys(0, 0);
  issue_values(0, 0);
  if (steps > 1) issue_keys(1, 1);

  // ---- this lane's query: chunks 2 f + kg
  uint4 qf[NF];
  {
    const bool have = pos < n && !a.q_zero;
    const T* row = (const T*)a.q + (int64_t)(start + (pos < n ? pos : 0)) * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int d = (2 * f + kg) * P::EPC;
      uint32_t w[4] = {0, 0, 0, 0};
      if (have && d < a.D) {
        if constexpr (VEC) {
          const uint4 x = *(const uint4*)(row + d);
          w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        } else {
#pragma unroll
          for (int e = 0; e < P::EPC; ++e)
            if (d + e < a.D) w[e * P::EB / 4] |= PElem<T>::bits(row + (int64_t)(d + e) * a.q_sd) << (8 * (e * P::EB % 4));
        }
      }
      qf[f] = make_uint4(w[0] ^ a.q_flip, w[1] ^ a.q_flip, w[2] ^ a.q_flip, w[3] ^ a.q_flip);
    }
  }

  // A wavefront's last tile holds its own positions; all before are seen whole.
  const int mine = first < n ? first / KT : -1;
  f32x16_t o[NDB];
  // A score's weight is exp2((s - base) * cs + neg): around the row's maximum m, which is kept in
  // the scores' own units. Up to kFar the maximum enters through neg, as one rounded product, which
  // saves the difference; beyond, that product's rounding (2^-24 of it) would pass what a weight's exponent
  // has room for, and base is the maximum itself, so that its weight is 2^bias whatever its size.
  constexpr float kFar = 65536.f;
  float m, neg, base, l;
  bool far;                                            // some row of the wavefront has a base
  const float cs = a.scale_log2;
  // How far above m a score may be. Finite, so that an overflowing difference is above it.
  const float slack = uniform(fminf(M::slack / cs, 3.4e38f));

  // One step of the first product over 32 keys at `kl`: register r of the scores is key
  // 8 (r / 4) + 4 kg + r % 4.
  const auto key_operand = [&](const unsigned char* kl, auto step) __attribute__((always_inline)) -> uint4 {
    return *(const uint4*)(kl + col * ROWB + P::k_place(col, 2 * decltype(step)::value + kg) * 16);
  };
  const auto score = [&](uint4 x, auto step, f32x16_t& s) __attribute__((always_inline)) {
    constexpr int f = decltype(step)::value;
    if constexpr (f == 0) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = 0.f;
    }
    if constexpr (P::F32) {
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.x), __uint_as_float(qf[f].x), s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.y), __uint_as_float(qf[f].y), s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.z), __uint_as_float(qf[f].z), s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.w), __uint_as_float(qf[f].w), s, 0, 0, 0);
    } else {
      s = M::mfma(x, qf[f], s);
    }
  };
  const auto mask = [&](int key0, f32x16_t& s) __attribute__((always_inline)) {
    int base = key0 + 4 * kg - pos;
    asm volatile("" : "+v"(base));  // defined here, so that no index arithmetic of this path is hoisted
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (base + 8 * (r / 4) + r % 4 > 0) s[r] = -INFINITY;
  };
  // Whether some row's running maximum moves with these scores; then `f` takes sums made with the old
  // one to the new (1 where it stays). Takes the base from the scores.
  const auto raise = [&](f32x16_t& s, float& f) __attribute__((always_inline)) -> bool {
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    const bool moves = __builtin_amdgcn_ballot_w64(top - m > slack) != 0;
    if (moves) {
      // Of the rows whose own scores ask for it: a row's bits are those of what it sees.
      const float both = fmaxf(top, __shfl_xor(top, 32, 64)), m2 = both - m > slack ? both : m, e = m2 * cs;
      const bool none = m2 == -INFINITY, away = !none && !(fabsf(e) <= kFar);
      const float base2 = away ? m2 : 0.f, neg2 = none ? 0.f : away ? M::bias : M::bias - e;
      f = m == -INFINITY ? 0.f : fast_exp2(__builtin_fmaf(base - base2, cs, neg2 - neg));
      m = m2, base = base2, neg = neg2;
      far = __builtin_amdgcn_ballot_w64(away) != 0;
      l *= f;
    }
    if (far) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] -= base;
    }
    return moves;
  };
  const auto scale_output = [&](float f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NDB; ++i) o[i] *= f;
  };
  // Weights of a 32-key block: element by element, then by pairs packed and summed.
  const auto weight = [&](f32x16_t& s, int r) __attribute__((always_inline)) {
    s[r] = fast_exp2(__builtin_fmaf(s[r], cs, neg));
  };
  const auto pack_pair = [&](const f32x16_t& s, int r, uint32_t (&w)[P::PREGS]) __attribute__((always_inline)) {
    if constexpr (P::F32) {
      l += s[2 * r] + s[2 * r + 1];
      w[2 * r] = __float_as_uint(s[2 * r]);
      w[2 * r + 1] = __float_as_uint(s[2 * r + 1]);
    } else {
      w[r] = M::pack2(s[2 * r], s[2 * r + 1]);
      l = M::sum2(w[r], l);
    }
  };
  const auto weights = [&](f32x16_t& s, uint32_t (&w)[P::PREGS]) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) weight(s, r);
#pragma unroll
    for (int r = 0; r < 8; ++r) pack_pair(s, r, w);
  };
  // One step of O^T += V^T P^T for 32 keys' values at `vl`: 16 keys and a block of dims (f32:
  // two keys). clean: what is not finite in V counts as 0.
  const int v_row = 4 * kg + ((lane & 15) >> 2);  // of 16 keys' first (and, + 8, second) 4-row piece
  const int v_c0 = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  constexpr int VSTEPS = P::F32 ? 16 * NDB : 2 * NDB;
  const auto value_operand = [&](const unsigned char* vl, auto step) __attribute__((always_inline)) -> uint4 {
    constexpr int n = decltype(step)::value, i = n % NDB, part = n / NDB;
    if constexpr (P::F32) {
      return make_uint4(*(const uint32_t*)(vl + (8 * (part / 4) + 4 * kg + part % 4) * ROWB + (32 * i + col) * 4), 0, 0, 0);
    } else {
      const uint32_t vb = lds_addr(vl) + v_row * ROWB + (lane & 1) * 8;
      const uint2 lo = TrRead<T>::at(vb + (16 * part) * ROWB + P::v_place(v_row, 4 * i + v_c0) * 16);
      const uint2 hi = TrRead<T>::at(vb + (16 * part + 8) * ROWB + P::v_place(v_row + 8, 4 * i + v_c0) * 16);
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  };
  const auto value = [&](uint4 x, auto step, const uint32_t (&w)[P::PREGS], auto clean) __attribute__((always_inline)) {
    constexpr int n = decltype(step)::value, i = n % NDB, part = n / NDB;
    if constexpr (decltype(clean)::value) x = make_uint4(P::finite(x.x), P::finite(x.y), P::finite(x.z), P::finite(x.w));
    if constexpr (P::F32)
      o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.x), __uint_as_float(w[part]), o[i], 0, 0, 0);
    else
      o[i] = M::mfma(x, make_uint4(w[4 * part], w[4 * part + 1], w[4 * part + 2], w[4 * part + 3]), o[i]);
  };
  const auto all_scores = [&](const unsigned char* kl, f32x16_t& s) __attribute__((always_inline)) {
    static_for<0, NF>([&](auto f) { score(key_operand(kl, f), f, s); });
  };
  const auto all_values = [&](const unsigned char* vl, const uint32_t (&w)[P::PREGS], auto clean) __attribute__((always_inline)) {
    static_for<0, VSTEPS>([&](auto n) { value(value_operand(vl, n), n, w, clean); });
  };
  const auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    m = -INFINITY, neg = 0.f, base = 0.f, l = 0.f, far = false;
  };
  f32x16_t sa, sb;
  uint32_t wa[P::PREGS], wb[P::PREGS];
  float f;

  // Three blocks of 32 keys are in work at once: block b's weights are made by the vector
  // units while the matrix cores make block b + 1's scores and add block b - 1's values,
  // and nothing among them waits for the others. So a tile's keys are needed a step before
  // its values, and are copied a step ahead of them.
  begin();
  wait_and_barrier<0>();
  const auto arrive = [&](int step, int buf) __attribute__((always_inline)) {
    wait_and_barrier<0>();  // the next keys and these values have landed, and the buffers below are done with
    if (step + 2 < steps) issue_keys(step + 2, buf);
    if (step + 1 < steps) issue_values(step + 1, buf ^ 1);
  };
  int step = 0;
  if constexpr (P::F32) {
    all_scores(k_lds[0], sa);
    const auto full = [&](int step, auto buf, f32x16_t& s, f32x16_t& next) __attribute__((always_inline)) {
      constexpr int B = decltype(buf)::value;
      arrive(step, B);
      if (raise(s, f)) scale_output(f);
      all_scores(k_lds[B ^ 1], next);
      weights(s, wa);
      all_values(v_lds[B], wa, std::false_type{});
    };
    for (; step + 1 < mine; step += 2) {
      full(step, Stage<0>{}, sa, sb);
      full(step + 1, Stage<1>{}, sb, sa);
    }
    if (step < mine) {
      full(step, Stage<0>{}, sa, sb);
      sa = sb;
      ++step;
    }
    if (mine >= 0) {
      arrive(step, step & 1);
      mask(step * KT, sa);
      if (raise(sa, f)) scale_output(f);
      weights(sa, wa);
      all_values(v_lds[step & 1], wa, std::false_type{});
      ++step;
    }
  } else {
    // Block b: weights of `s` into `w`, beside the next block's scores (NEXT), the last one's
    // values, and the copies of a later tile of keys and of values (COPY), which would hold
    // the wavefront up for about 100 cycles each if they were issued one after the other.
    const char *k_from = nullptr, *v_from = nullptr;
    const auto block = [&](int b, const unsigned char* kl, const unsigned char* vl, f32x16_t& s, f32x16_t& next,
                           const uint32_t (&before)[P::PREGS], uint32_t (&w)[P::PREGS], auto has_next, auto copy,
                           uint32_t copy_to) __attribute__((always_inline)) {
      constexpr bool NEXT = decltype(has_next)::value;
      constexpr int COPY = decltype(copy)::value;  // 0: none, 1: keys, 2: values
      // Operands are read LEAD steps ahead, the first before the maximum.
      constexpr int LEAD = 2, KSTEPS = NEXT ? NF : 0, SLOTS = KSTEPS + VSTEPS, EACH = (16 + SLOTS - 1) / SLOTS;
      constexpr int LONG = KSTEPS > VSTEPS ? KSTEPS : VSTEPS;
      uint4 kx[NF], vx[VSTEPS];
      static_for<0, LEAD>([&](auto i) {
        constexpr int n = decltype(i)::value;
        if constexpr (n < KSTEPS) kx[n] = key_operand(kl, i);
        if constexpr (n < VSTEPS) vx[n] = value_operand(vl, i);
      });
      __builtin_amdgcn_sched_barrier(0);
      if (COPY == 0 && b >= 2 * mine) mask(32 * b, s);
      const bool raised = raise(s, f);
      // Each product is followed by its share of the weights, in this order.
      const auto share = [&](auto slot) __attribute__((always_inline)) {
        constexpr int n = decltype(slot)::value;
#pragma unroll
        for (int r = n * EACH; r < (n + 1) * EACH && r < 16; ++r) {
          weight(s, r);
          if (r >= 3 && r % 2 == 1) pack_pair(s, r / 2 - 1, w);
        }
        if constexpr (COPY != 0) {
          constexpr int GAP = SLOTS / P::COPIES;
          if constexpr (n % GAP == 0 && n / GAP < P::COPIES) {
            if constexpr (COPY == 1) P::template copy_piece<true, n / GAP>(a, k_from, a.k_st, copy_to);
            else P::template copy_piece<false, n / GAP>(a, v_from, a.v_st, copy_to);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, LONG>([&](auto i) {
        constexpr int n = decltype(i)::value;
        if constexpr (n + LEAD < KSTEPS) kx[n + LEAD] = key_operand(kl, Stage<n + LEAD>{});
        if constexpr (n < KSTEPS) {
          score(kx[n], i, next);
          share(Stage<n + (n < VSTEPS ? n : VSTEPS)>{});
        }
        if constexpr (n + LEAD < VSTEPS) vx[n + LEAD] = value_operand(vl, Stage<n + LEAD>{});
        if constexpr (n < VSTEPS) {
          value(vx[n], i, before, std::false_type{});
          share(Stage<n + (n + 1 < KSTEPS ? n + 1 : KSTEPS)>{});
        }
      });
      pack_pair(s, 7, w);
      // Made here, not where they are first used, behind the branch below.
      asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]), "+v"(w[4]), "+v"(w[5]), "+v"(w[6]), "+v"(w[7]), "+v"(l));
      __builtin_amdgcn_sched_barrier(0);
      if (raised) scale_output(f);
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    // In the middle of a long prompt: two whole tiles to copy, and nothing to mask.
    const int middle = VEC && a.D == DP ? min(min(mine - 1, steps - 2), n / KT - 2) : 0;  // steps below it
    const auto full = [&](int step, auto buf) __attribute__((always_inline)) {
      constexpr int B = decltype(buf)::value;
      wait_and_barrier<0>();
      k_from = (const char*)(kh + (int64_t)(step + 2) * KT * a.k_st);
      v_from = (const char*)(vh + (int64_t)(step + 1) * KT * a.v_st);
      block(2 * step + 1, k_lds[B ^ 1], v_lds[B], sa, sb, wa, wb, yes, Stage<2>{}, lds_addr(v_lds[B ^ 1]));
      block(2 * step + 2, k_lds[B ^ 1] + 32 * ROWB, v_lds[B] + 32 * ROWB, sb, sa, wb, wa, yes, Stage<1>{}, lds_addr(k_lds[B]));
    };
    // Block 0: its weights beside block 1's scores.
    all_scores(k_lds[0], sb);
    all_scores(k_lds[0] + 32 * ROWB, sa);
    if (mine == 0) mask(0, sb);
    raise(sb, f);
    weights(sb, wa);
    for (; step + 1 < middle; step += 2) {
      full(step, Stage<0>{});
      full(step + 1, Stage<1>{});
    }
#pragma unroll 1
    for (; step < mine; ++step) {
      const int buf = step & 1;
      arrive(step, buf);
      const unsigned char *kl = k_lds[buf ^ 1], *vl = v_lds[buf];
      block(2 * step + 1, kl, vl, sa, sb, wa, wb, yes, Stage<0>{}, 0);
      block(2 * step + 2, kl + 32 * ROWB, vl + 32 * ROWB, sb, sa, wb, wa, yes, Stage<0>{}, 0);
    }
    if (mine >= 0) {
      arrive(step, step & 1);
      if (64 * step + 32 <= last) {
        block(2 * step + 1, nullptr, v_lds[step & 1], sa, sb, wa, wb, no, Stage<0>{}, 0);
        all_values(v_lds[step & 1] + 32 * ROWB, wb, no);
      } else {  // the tile's second half lies behind this wavefront's rows
        all_values(v_lds[step & 1], wa, no);
      }
      ++step;
    }
  }
  for (; step < steps; ++step) arrive(step, step & 1);

  // With a masked weight of 0, an infinity or a NaN in a value that a row does not see
  // still makes a NaN of it in the matrix product. That shows in the output; then the
  // workgroup goes over its tiles again, with such values taken out of the product and
  // added to the rows that see them.
  float lost = l * 0.f;
#pragma unroll
  for (int i = 0; i < NDB; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) lost = __builtin_fmaf(o[i][j], 0.f, lost);
  if (__syncthreads_or(pos < n && lost != lost)) {
    begin();
#pragma unroll 1
    for (step = 0; step < steps; ++step) {
      __syncthreads();
      issue_keys(step, 0);
      issue_values(step, 0);
      wait_and_barrier<0>();
      if (step > mine) continue;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        all_scores(k_lds[0] + kb * 32 * ROWB, sa);
        mask(step * KT + 32 * kb, sa);
        if (raise(sa, f)) scale_output(f);
        weights(sa, wa);
        all_values(v_lds[0] + kb * 32 * ROWB, wa, std::true_type{});
      }
#pragma unroll 1
      for (int key = 0; key < KT; ++key) {
        const bool seen = step * KT + key <= pos;
#pragma unroll
        for (int i = 0; i < NDB; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int d = 32 * i + 8 * j + 4 * kg;
            const unsigned char* at = v_lds[0] + key * ROWB + P::v_place(key, d / P::EPC) * 16 + d % P::EPC * P::EB;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = Elem<T>::load((const T*)at + e);
              if (seen && !(fabsf(x) < INFINITY)) o[i][4 * j + e] += x;
            }
          }
      }
    }
    __syncthreads();  // the output goes through these tiles
  }

  // ---- out: registers 4 j .. 4 j + 3 of block i are dims 32 i + 8 j + 4 kg .. of row `pos`
  const float total = l + __shfl_xor(l, 32, 64), inv = total == 0.f ? 0.f : 1.f / total;
  if constexpr (VEC) {
    // Through LDS, which no wavefront reads any more: whole rows leave in 16-byte pieces
    // (3k cycles; straight from the registers, 8-byte pieces of 32 rows a store, 5k).
    unsigned char* mine_lds = &k_lds[0][0] + wave * (32 * ROWB);  // k_lds and v_lds hold 128 rows and more
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x0 = o[i][4 * j] * inv, x1 = o[i][4 * j + 1] * inv, x2 = o[i][4 * j + 2] * inv, x3 = o[i][4 * j + 3] * inv;
        const int d = 32 * i + 8 * j + 4 * kg;
        unsigned char* at = mine_lds + col * ROWB + P::k_place(col, d / P::EPC) * 16 + d % P::EPC * P::EB;
        if constexpr (P::F32) *(float4*)at = make_float4(x0, x1, x2, x3);
        else *(uint2*)at = make_uint2(M::pack2(x0, x1), M::pack2(x2, x3));
      }
    __builtin_amdgcn_wave_barrier();
    T* out = (T*)a.out + (int64_t)(start + first) * a.o_st + (int64_t)h * a.o_sh;
#pragma unroll
    for (int i = 0; i < 32 * P::CPR / 64; ++i) {
      const int at = i * 64 + lane, row = at / P::CPR, c = at % P::CPR;
      const uint4 x = *(const uint4*)(mine_lds + row * ROWB + P::k_place(row, c) * 16);
      if (first + row < n && c * P::EPC < a.D) *(uint4*)(out + (int64_t)row * a.o_st + c * P::EPC) = x;
    }
  } else if (pos < n) {
    T* row = (T*)a.out + (int64_t)(start + pos) * a.o_st + (int64_t)h * a.o_sh;
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int d = 32 * i + 8 * (j / 4) + 4 * kg + j % 4;
        if (d < a.D) Elem<T>::store(row + d * a.o_sd, o[i][j] * inv);
      }
  }
}

template <typename T, int DP>
hipError_t launch_prompt_dp(PromptArgs a, hipStream_t stream) {
  const int rows = kPromptRows / a.heads;
  const int64_t tiles = (int64_t)a.T / rows + std::min<int64_t>(a.B, a.T);
  const int64_t grid = std::max<int64_t>(1, tiles * (a.Hq / a.heads));
  void* args[] = {&a};
  const void* fn = a.vec ? (const void*)&prompt_attention_kernel<T, DP, true> : (const void*)&prompt_attention_kernel<T, DP, false>;
  return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(256), args, 0, stream);
}

template <typename T>
hipError_t launch_prompt(const PromptArgs& a, hipStream_t stream) {
  if (a.D <= 32) return launch_prompt_dp<T, 32>(a, stream);
  if (a.D <= 64) return launch_prompt_dp<T, 64>(a, stream);
  if (a.D <= 80) return launch_prompt_dp<T, 80>(a, stream);
  if (a.D <= 96) return launch_prompt_dp<T, 96>(a, stream);
  if (a.D <= 128) return launch_prompt_dp<T, 128>(a, stream);
  if (a.D <= 192) return launch_prompt_dp<T, 192>(a, stream);
  if (a.D <= 256) return launch_prompt_dp<T, 256>(a, stream);
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace mgi
