// paged_fp4.h -- decode attention over the 4-bit paged pool (fp4_kv.h), one query token
// per sequence, grouped query heads.
//
//   out[b,h] = sum_t softmax_t(scale * q[b,h] . K[t, h / G]) V[t, h / G],  t < ctx[b]
//
// What it has to read is 34 bytes per 64 cached values; per KV head and token that is 136
// bytes at D = 128 for 4 G D flops, so it is bound by memory, and the work is to undo the
// codes with few enough instructions to keep up. gfx950 converts a byte of codes and its
// group's scale to two bf16 in one instruction (exactly: a code has two significant bits),
// and the products run on the matrix cores:
//   S^T[16 tokens, 16 queries] = K Q^T,   O^T[dims, 16 queries] += V^T P^T
// with 16x16x32 bf16 MFMAs, a tile of 32 tokens at a time per wavefront. A lane's column is
// one query head, so the softmax's running maximum and sum are its own, and S^T's layout
// (lane: query l % 16, tokens 4 (l / 16) .. + 3 of each 16) is the layout P^T needs when
// the tokens of V are taken in the same order: no value crosses lanes but the maxima.
// Keys: a lane's codes are 16 consecutive bytes of one token's row, one group. Values: a
// lane's codes are the dims that are its row of V^T, for its 8 tokens.
//
// Measured on MI355X, D = 128, bf16, where a large copy reaches 5.05 TB/s: 64 sequences of 512-4096
// tokens, 32 heads, 132 us (5.2 TB/s); 8 of 32k-128k, 32 heads on 8, 174 us (5.4 TB/s); 13 of
// 100-1000, 16 heads, 11 us; 256 of 128-2048, 32 heads of 64 on 8, f16, 57 us (2.5 TB/s: up to 8
// tiles a wavefront, whose chains of table entry, codes and products nothing hides).
// Of a large call's wavefront cycles half are waits, 42 % have a vector instruction in work.
//
// Numerics: q is cut into bf16 terms that add up to it (1 for bf16, 2 for f16, 3 for f32; what an
// f32 element has below 2^-133, bf16's least number, is left out), so scores are f32 sums of exact products. The softmax weights are cut into 2 terms (3 for
// f32 outputs), 2^-17 (2^-26) of a weight at most, where one term would cost 2^-8: the
// matrix cores have the room, as 4-bit keys and values arrive slower than they multiply.
// A weight's exponent is (score - maximum) * scale, the difference first: a product of each
// would round by 2^-24 of itself, which overflows weights of scores far from 0.
#pragma once

#include <type_traits>

#include "fp4_kv.h"
#include "minivllm_hip.h"

namespace mgi {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;          // tokens per step of a wavefront
constexpr float kNoMax = -3.4028234e38f;  // no score yet: the lowest finite number, so that differences are no NaN

// A row of NG groups is handled in pieces of 4, 2 or 1 groups, so that a lane's share of a
// piece is a power of two: piece p starts at group start(p) and has size(p) groups.
template <int NG> struct Pieces {
  static constexpr int count = NG / 4 + ((NG >> 1) & 1) + (NG & 1);
  static constexpr int size(int p) {
    if (p < NG / 4) return 4;
    return p == NG / 4 && (NG & 2) ? 2 : 1;
  }
  static constexpr int start(int p) {
    int at = 0;
    for (int i = 0; i < p; ++i) at += size(i);
    return at;
  }
};

template <typename T> struct Terms;  // bf16 terms of a query element and of a softmax weight
template <> struct Terms<bf16_t> { static constexpr int q = fp4_query_terms(2, true), p = 2; };
template <> struct Terms<f16_t> { static constexpr int q = fp4_query_terms(2, false), p = 2; };
template <> struct Terms<float> { static constexpr int q = fp4_query_terms(4, false), p = 3; };

// A stride whose products the compiler does not compute ahead of the loop over (sequence,
// head) pairs, where they would take a hundred registers.
__device__ __forceinline__ int64_t unhoisted(int64_t x) {
  asm volatile("" : "+s"(x));
  return x;
}

template <int I> using Int = std::integral_constant<int, I>;
template <int B, int E, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (B < E) {
    f(Int<B>{});
    each<B + 1, E>(f);
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const f32x2_t x = {lo, hi};  // converted as a vector: one instruction (three, element by element)
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2_t));
}
__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}
template <int BYTE>
__device__ __forceinline__ uint32_t two_bf16(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
}

__device__ __forceinline__ float across_max(float x) {  // over the four lanes of a query
  x = fmaxf(x, swizzle_xor16(x));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float across_sum(float x) {
  x += swizzle_xor16(x);
  return x + __shfl_xor(x, 32, 64);
}

__device__ __forceinline__ int context_of(const Fp4DecodeArgs& a, int b) {
  const int64_t c = load_index(a.cl, a.cl_i64, (int64_t)b * a.cl_s), most = (int64_t)a.M * a.S;
  return (int)(c < 0 ? 0 : c > most ? most : c);
}

// One (sequence, KV head, query tile): its queries, running softmax and output.
template <typename T, int NG, bool ANY>
struct Attend {
  using P = Pieces<NG>;
  static constexpr int NQ = Terms<T>::q, NP = Terms<T>::p;

  // Where 32 tokens are: the slabs and offsets of each 16 (ANY: of token l % 16 of them).
  struct Place {
    const unsigned char* slab[2];
    uint32_t off[2];
    uint32_t valid;             // bit t: token t is in the context and its block is in the pool
  };
  // Their codes and scales: 16 + 16 rows of keys, 8 tokens' values.
  struct Keys {
    uint32_t w[2][NG];          // words of the lane's 16-token row, piece by piece
    uint32_t s[2][P::count];    // its group's byte
  };
  struct Values {
    uint32_t w[8][P::count];    // the lane's dims of its tokens 0..3 and 16..19 (+ 4 (l / 16))
    uint32_t s[2][P::count];    // four tokens' bytes
  };

  const Fp4DecodeArgs& a;
  int lane, c, kg;              // c: query, key row, or dims of V^T; kg: which of the four lanes
  const unsigned char* head;    // the pool at this KV head
  const char* table;            // the sequence's row of the block table
  int ctx;
  u32x4_t q[NQ][NG];
  f32x4_t acc[2 * NG];
  float m, l;                   // maximum, in the scores' own units (before the scale), and sum
  int entries, entries_at;      // block ids of 64 subtiles from subtile `entries_at` on, one per lane

  __device__ __forceinline__ Attend(const Fp4DecodeArgs& args)
      : a(args) {}

  __device__ __forceinline__ int64_t entry(int blk) const {
    const int64_t e = load_index(table, a.bt_i64, (int64_t)blk * a.bt_sm);
    return e < 0 || e >= a.N ? -1 : e;
  }

  // Queries of heads hq0 .. hq0 + 15 (fewer at the end of the group), as bf16 terms.
  __device__ __forceinline__ void begin(int b, int hk, int qt, int context) {
    // Defined anew, so that addresses made of them are not kept over the loop over pairs.
    lane = (int)(threadIdx.x & 63);
    asm volatile("" : "+v"(lane));
    c = lane & 15, kg = lane >> 4;
    ctx = context;
    head = a.pool + hk * a.p_sh;
    table = (const char*)a.bt + ((int64_t)b * a.bt_sb) * (a.bt_i64 ? 8 : 4);
    m = kNoMax;
    l = 0.f;
    entries_at = -(1 << 30);
#pragma unroll
    for (int j = 0; j < 2 * NG; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int g = qt * 16 + c;
    const bool have = g < a.G && !a.q_zero;
    const T* row = (const T*)a.q + (int64_t)b * a.q_sb + (int64_t)(hk * a.G + (have ? g : 0)) * a.q_sh;
    each<0, P::count>([&](auto pc) {
      constexpr int s = P::size(pc), g0 = P::start(pc);
      each<0, s>([&](auto i) {
        const int d0 = g0 * 32 + (kg * s + i) * 8;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
        if (have && d0 < a.D) {
          if (a.vec) {
            if constexpr (sizeof(T) == 4) {
              const float4 u = *(const float4*)(row + d0), w = *(const float4*)(row + d0 + 4);
              x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
            } else {
              const uint4 u = *(const uint4*)(row + d0);
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                T t;
                t.bits = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
                x[e] = Elem<T>::load(&t);
              }
            }
          } else {
            const int64_t sd = unhoisted(a.q_sd);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (d0 + e < a.D) x[e] = Elem<T>::load(row + (d0 + e) * sd);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(__float_as_uint(x[e]) ^ a.q_flip);
        }
        each<0, NQ>([&](auto n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w;
            if constexpr (NQ == 3)  // cut off: three times 8 bits are all 24, and the largest numbers stay finite
              w = __builtin_amdgcn_perm(__float_as_uint(x[2 * e + 1]), __float_as_uint(x[2 * e]), 0x07060302u);
            else
              w = pack_bf16(x[2 * e], x[2 * e + 1]);
            q[n][g0 + i][e] = w;
            x[2 * e] -= bf16_lo(w);
            x[2 * e + 1] -= bf16_hi(w);
          }
        });
      });
    });
  }

  __device__ __forceinline__ static uint32_t load32(const unsigned char* p) {
    return __builtin_nontemporal_load((const uint32_t*)p);
  }

  template <int PC>
  __device__ __forceinline__ static uint32_t load_v(const unsigned char* p) {  // size(PC) bytes
    if constexpr (P::size(PC) == 4) return __builtin_nontemporal_load((const uint32_t*)p);
    else if constexpr (P::size(PC) == 2) return __builtin_nontemporal_load((const uint16_t*)p);
    else return __builtin_nontemporal_load(p);
  }

  template <int PC>
  __device__ __forceinline__ static void load_k(uint32_t* dst, const unsigned char* p) {
    constexpr int s = P::size(PC);
    if constexpr (s == 4) {
      const u32x4_t w = __builtin_nontemporal_load((const u32x4_t*)p);
      dst[0] = w[0], dst[1] = w[1], dst[2] = w[2], dst[3] = w[3];
    } else if constexpr (s == 2) {
      const u32x2_t w = __builtin_nontemporal_load((const u32x2_t*)p);
      dst[0] = w[0], dst[1] = w[1];
    } else {
      dst[0] = load32(p);
    }
  }

  // Tokens 32 * tile .. + 31. A token past the context, or in a block outside the pool, is given
  // a place in block 0, so that every address is inside the pool.
  __device__ __forceinline__ Place find(int tile) {
    Place t;
    const int S = a.S;
    t.valid = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (!ANY) {  // S is a multiple of 16: 16 tokens lie in one block
        const int sub = 2 * tile + j, tok = sub * 16;
        if (sub - entries_at >= 64) {
          entries_at = sub;
          const int mine = (sub + lane) * 16;
          entries = mine < ctx ? (int)entry(fast_div(mine, a.s_mul, a.s_shift, S)) : -1;
        }
        const int phys = __builtin_amdgcn_readlane(entries, sub - entries_at);
        const int blk = fast_div(tok, a.s_mul, a.s_shift, S);
        t.off[j] = (uint32_t)__builtin_amdgcn_readfirstlane(tok - blk * S);
        const int left = phys < 0 ? 0 : min(16, ctx - tok);
        t.valid |= (left <= 0 ? 0u : 0xffffu >> (16 - left)) << (16 * j);
        t.slab[j] = head + (int64_t)(phys < 0 ? 0 : phys) * a.p_sn;
      } else {
        const int tok = 32 * tile + 16 * j + c;
        const int blk = fast_div(tok, a.s_mul, a.s_shift, S);
        const int64_t phys = tok < ctx ? entry(blk) : -1;
        t.off[j] = phys < 0 ? 0u : (uint32_t)(tok - blk * S);
        t.valid |= (uint32_t)(__ballot(phys >= 0) & 0xffffu) << (16 * j);
        t.slab[j] = head + (phys < 0 ? 0 : phys) * a.p_sn;
      }
    }
    return t;
  }

  __device__ __forceinline__ void load(Keys& k, const Place& t) {
    const uint32_t ks = fp4_k_scales(a.S, NG);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      each<0, P::count>([&](auto pc) {
        constexpr int s = P::size(pc), g0 = P::start(pc);
        const int row = ANY ? 0 : c;  // behind the place
        load_k<pc>(&k.w[j][g0], t.slab[j] + t.off[j] * (NG * 16) + g0 * 16 + (uint32_t)(row * (NG * 16) + kg * (s * 4)));
        k.s[j][pc] = __builtin_nontemporal_load(t.slab[j] + ks + t.off[j] * NG + g0 + (uint32_t)(row * NG + kg * s / 4));
      });
  }

  __device__ __forceinline__ void load(Values& v, const Place& t) {
    const uint32_t S = a.S, vc = fp4_v_codes(S, NG), vs = fp4_v_scales(S, NG);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (!ANY) {
        each<0, P::count>([&](auto pc) {
          constexpr int s = P::size(pc), g0 = P::start(pc);
          const unsigned char* vb = t.slab[j] + vc + t.off[j] * (NG * 16) + g0 * 16;
          each<0, 4>([&](auto i) {
            v.w[4 * j + i][pc] = load_v<pc>(vb + i * (NG * 16) + (uint32_t)(kg * 4 * (NG * 16) + c * s));
          });
          v.s[j][pc] = load32(t.slab[j] + vs + g0 * S + t.off[j] + (uint32_t)(c * s / 16 * S + kg * 4));
        });
      } else {
        const uint64_t base = (uint64_t)t.slab[j];
        each<0, P::count>([&](auto pc) { v.s[j][pc] = 0; });
        each<0, 4>([&](auto i) {  // lane t (< 16) knows token t's place
          const int from = kg * 4 + i;
          const unsigned char* slab = (const unsigned char*)(((uint64_t)(uint32_t)__shfl((int)(base >> 32), from, 64) << 32) |
                                                             (uint32_t)__shfl((int)base, from, 64));
          const uint32_t off = (uint32_t)__shfl((int)t.off[j], from, 64);
          each<0, P::count>([&](auto pc) {
            constexpr int s = P::size(pc), g0 = P::start(pc);
            v.w[4 * j + i][pc] = load_v<pc>(slab + vc + off * (NG * 16) + g0 * 16 + (uint32_t)(c * s));
            v.s[j][pc] |= (uint32_t)slab[vs + (g0 + c * s / 16) * S + off] << (8 * i);
          });
        });
      }
    }
  }

  // Scores: rows 4 kg .. + 3 of each 16 tokens, column c.
  __device__ __forceinline__ void scores(const Keys& k, float (&s)[8]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4_t r = {0.f, 0.f, 0.f, 0.f};
      each<0, P::count>([&](auto pc) {
        constexpr int sz = P::size(pc), g0 = P::start(pc);
        const float scale = __uint_as_float(k.s[j][pc] << 23);
        each<0, sz>([&](auto i) {
          const uint32_t w = k.w[j][g0 + i];
          const u32x4_t x = {two_bf16<0>(w, scale), two_bf16<1>(w, scale), two_bf16<2>(w, scale), two_bf16<3>(w, scale)};
          each<0, NQ>([&](auto n) { r = mfma(x, q[n][g0 + i], r); });
        });
      });
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * j + i] = r[i];
    }
  }

  // Softmax weights of the scores, as bf16 terms; masked tokens' values are made finite. Weights
  // carry a factor of 2^-kFp4Slack, so that no sum of them times values passes the softmax's.
  __device__ __forceinline__ void weights(float (&s)[8], uint32_t valid, Values& v, u32x4_t (&w)[NP]) {
    if (valid != 0xffffffffu) {  // the end of the context, or a block outside the pool
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = (valid >> (16 * (i / 4) + kg * 4 + i % 4)) & 1;
        s[i] = in ? s[i] : -INFINITY;
        // What stands in a masked place has weight 0, and must not be NaN.
        each<0, P::count>([&](auto pc) {
          if (!in) v.s[i / 4][pc] = (v.s[i / 4][pc] & ~(0xffu << (8 * (i % 4)))) | (127u << (8 * (i % 4)));
        });
      }
    }
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    if (__any(top - m > a.slack)) {
      const float m2 = fmaxf(m, across_max(top)), f = fast_exp2((m - m2) * a.scale_log2);
      m = m2;
      l *= f;
#pragma unroll
      for (int j = 0; j < 2 * NG; ++j) acc[j] *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = fast_exp2(__builtin_fmaf(s[i] - m, a.scale_log2, -kFp4Slack));
    l += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    each<0, NP>([&](auto n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[n][e] = pack_bf16(s[2 * e], s[2 * e + 1]);
        s[2 * e] -= bf16_lo(w[n][e]);
        s[2 * e + 1] -= bf16_hi(w[n][e]);
      }
    });
  }

  __device__ __forceinline__ void add(const Values& v, const u32x4_t (&w)[NP]) {
    each<0, P::count>([&](auto pc) {
      constexpr int sz = P::size(pc), g0 = P::start(pc);
      float scale[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) scale[i] = __uint_as_float(((v.s[i / 4][pc] >> (8 * (i % 4))) & 0xffu) << 23);
      each<0, sz>([&](auto b) {  // byte b: dims 2 b and 2 b + 1 of the lane's
        u32x4_t even, odd;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = two_bf16<b>(v.w[2 * e][pc], scale[2 * e]), y = two_bf16<b>(v.w[2 * e + 1][pc], scale[2 * e + 1]);
          even[e] = __builtin_amdgcn_perm(y, x, 0x05040100u);
          odd[e] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        }
        each<0, NP>([&](auto n) {
          acc[2 * (g0 + b)] = mfma(even, w[n], acc[2 * (g0 + b)]);
          acc[2 * (g0 + b) + 1] = mfma(odd, w[n], acc[2 * (g0 + b) + 1]);
        });
      });
    });
  }

  // Tiles first, first + step, .. below end. A tile's keys are asked for when the last one's have
  // been multiplied, its values when the last one's have been: one set of registers of each,
  // and four wavefronts to a SIMD, whose loads are in flight while others compute.
  __device__ __forceinline__ void run(int first, int end, int step) {
    if (first >= end) return;
    Keys k;
    Values v;
    Place t = find(first);
    load(k, t);
    load(v, t);
    for (int tile = first; tile < end; tile += step) {
      const uint32_t valid = t.valid;
      float s[8];
      scores(k, s);
      const bool more = tile + step < end;
      if (more) {
        t = find(tile + step);
        load(k, t);
      }
      u32x4_t w[NP];
      weights(s, valid, v, w);
      add(v, w);
      if (more) load(v, t);
    }
  }

  // Calls f(dim, four values) for the lane's dims of query c (dims of a piece: 8 size
  // consecutive ones from start * 32 + kg * 8 size on).
  template <typename F>
  __device__ __forceinline__ void dims(F&& f) const {
    each<0, P::count>([&](auto pc) {
      constexpr int s = P::size(pc), g0 = P::start(pc);
      each<0, 2 * s>([&](auto e) {
        // Values 4 e .. 4 e + 3 of the 8 s: value v is accumulator v % (2 s), row v / (2 s).
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          constexpr int width = 2 * s;
          x[i] = acc[2 * g0 + (4 * e + i) % width][(4 * e + i) / width];
        }
        f(g0 * 32 + kg * (8 * s) + 4 * e, x[0], x[1], x[2], x[3]);
      });
    });
  }
};

// Four neighbouring dims of an output row.
template <typename T>
__device__ __forceinline__ void store4(const Fp4DecodeArgs& a, T* row, int d, float x0, float x1, float x2, float x3) {
  const float x[4] = {x0, x1, x2, x3};
  if (a.vec) {
    if (d >= a.D) return;
    if constexpr (sizeof(T) == 4) {
      *(float4*)(row + d) = make_float4(x0, x1, x2, x3);
    } else {
      T e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) Elem<T>::store(&e[i], x[i]);
      *(uint2*)(row + d) = make_uint2((uint32_t)e[0].bits | ((uint32_t)e[1].bits << 16),
                                      (uint32_t)e[2].bits | ((uint32_t)e[3].bits << 16));
    }
  } else {
    const int64_t sd = unhoisted(a.o_sd);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < a.D) Elem<T>::store(row + (d + i) * sd, x[i]);
  }
}

template <typename T>
__device__ __forceinline__ T* out_row(const Fp4DecodeArgs& a, int b, int h) {
  return (T*)a.out + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh;
}

// 1 / sum of weights; 0 for a row without keys.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// The whole call in one launch: a workgroup per (sequence, KV head, query tile), whose
// wavefronts take its tiles in turn and meet in LDS.
template <typename T, int NG, bool ANY>
__global__ void __launch_bounds__((64 * fp4_one_waves(NG, Terms<T>::q))) paged_fp4_one(const Fp4DecodeArgs a) {
  extern __shared__ float lds[];
  const int waves = (int)(blockDim.x >> 6), wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.Hk * a.q_tiles, b = (int)blockIdx.x / heads, r = (int)blockIdx.x - b * heads;
  const int hk = r / a.q_tiles, qt = r - hk * a.q_tiles;
  const int ctx = __builtin_amdgcn_readfirstlane(context_of(a, b));
  const int rows = min(16, a.G - qt * 16);
  Attend<T, NG, ANY> at(a);
  at.begin(b, hk, qt, ctx);
  at.run(wave, (ctx + kTile - 1) / kTile, waves);
  // [wave][row]: dims, then the maximum and the sum.
  constexpr int width = NG * 32 + 4;
  const float l = across_sum(at.l);
  if (at.c < rows) {
    float* row = lds + (wave * rows + at.c) * width;
    at.dims([&](int d, float x0, float x1, float x2, float x3) { *(float4*)(row + d) = make_float4(x0, x1, x2, x3); });
    if (at.kg == 0) row[NG * 32] = at.m, row[NG * 32 + 1] = l;
  }
  __syncthreads();
  for (int i = (int)threadIdx.x; i < rows * NG * 8; i += (int)blockDim.x) {
    const int row = i / (NG * 8), d = (i - row * (NG * 8)) * 4;
    float m = kNoMax, sum = 0.f;
    for (int w = 0; w < waves; ++w) m = fmaxf(m, lds[(w * rows + row) * width + NG * 32]);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < waves; ++w) {
      const float* part = lds + (w * rows + row) * width;
      const float f = fast_exp2((part[NG * 32] - m) * a.scale_log2);
      const float4 y = *(const float4*)(part + d);
      sum += f * part[NG * 32 + 1];
      x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
    }
    const float inv = inverse(sum);
    store4(a, out_row<T>(a, b, hk * a.G + qt * 16 + row), d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  }
}

// Tiles of all (sequence, KV head, query tile), in that order, cut into runs that differ by
// one tile at most, one per wavefront: as many as are resident at once. A (sequence, head)
// inside one run is finished by it; the others leave (maximum, sum, unnormalised output) for
// paged_fp4_join: slot 2 w for a run's beginning inside a (sequence, head), 2 w + 1 for its
// end. A run has kShortestRun tiles or more (or all), so that little is left to join: with
// runs of one tile, and a join of one wavefront, 2 sequences of 8k tokens on 2 KV heads took
// 82 us, with this 18. Runs of 2 tiles or more: 1-3 us less on few rows of 1k-8k, 6 more on one
// of 32k; of 8: 1-5 more on all of them.
constexpr int kShortestRun = 4;
struct Runs {
  int64_t size, longer;  // tiles of a run; so many first runs have one more
  int count;
  __device__ __forceinline__ Runs(int64_t total, int waves)
      : count((int)max((int64_t)1, min((int64_t)waves, total / kShortestRun))) {
    size = total / count;
    longer = total - size * count;
  }
  __device__ __forceinline__ int64_t start(int w) const { return size * w + (w < longer ? w : longer); }
  __device__ __forceinline__ int of(int64_t pos) const {  // the run with tile pos
    const int64_t at = longer * (size + 1);
    return (int)(pos < at ? pos / (size + 1) : longer + (pos - at) / size);
  }
};

template <typename T, int NG, bool ANY>
__global__ void __launch_bounds__(256, (fp4_occupancy(NG, Terms<T>::q))) paged_fp4_split(const Fp4DecodeArgs a) {
  const int wave = (int)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int lane = (int)(threadIdx.x & 63), heads = a.Hk * a.q_tiles;
  // All tiles of one head, and from them this wavefront's run.
  int sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) sum += b0 + lane < a.B ? (context_of(a, b0 + lane) + kTile - 1) / kTile : 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
  const int tiles = __builtin_amdgcn_readfirstlane(sum);
  const int64_t total = (int64_t)tiles * heads;
  const Runs runs(total, a.waves);
  const int64_t start = runs.start(wave);
  int64_t left = wave < runs.count ? runs.start(wave + 1) - start : 0;
  if (left <= 0 && wave != 0) return;
  // The sequence the run starts in: the first whose tiles, with those before it, pass start / heads.
  const int want = (int)(start / heads);
  int b = -1, b_before = 0, before = 0;
  for (int b0 = 0; b0 < a.B && (b < 0 || wave == 0); b0 += 64) {
    const int n = b0 + lane < a.B ? (context_of(a, b0 + lane) + kTile - 1) / kTile : 0;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(upto, d, 64);
      if (lane >= d) upto += y;
    }
    if (wave == 0 && b0 + lane < a.B) a.ws_cum[b0 + lane] = before + upto - n;
    const uint64_t past = __ballot(before + upto > want);
    if (b < 0 && past) {
      const int i = __ffsll((unsigned long long)past) - 1;
      b = b0 + i;
      b_before = before + __builtin_amdgcn_readlane(upto - n, i);
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  if (wave == 0 && lane == 0) a.ws_cum[a.B] = tiles;
  if (left <= 0) return;
  int ctx = __builtin_amdgcn_readfirstlane(context_of(a, b)), n = (ctx + kTile - 1) / kTile;
  const int64_t in = start - (int64_t)b_before * heads;
  int r = __builtin_amdgcn_readfirstlane((int)(in / n)), first = __builtin_amdgcn_readfirstlane((int)(in - (int64_t)r * n));
  Attend<T, NG, ANY> at(a);
  while (true) {
    const int last = (int)min((int64_t)n, first + left);
    const int hk = r / a.q_tiles, qt = r - hk * a.q_tiles, rows = min(16, a.G - qt * 16);
    at.begin(b, hk, qt, ctx);
    at.run(first, last, 1);
    left -= last - first;
    const float l = across_sum(at.l);
    if (at.c < rows) {
      if (first == 0 && last == n) {
        const float inv = inverse(l);
        T* row = out_row<T>(a, b, hk * a.G + qt * 16 + at.c);
        at.dims([&](int d, float x0, float x1, float x2, float x3) {
          store4(a, row, d, x0 * inv, x1 * inv, x2 * inv, x3 * inv);
        });
      } else {
        const int64_t slot = 2 * (int64_t)wave + (first == 0);
        float* row = a.ws_acc + (slot * min(a.G, 16) + at.c) * (NG * 32);
        at.dims([&](int d, float x0, float x1, float x2, float x3) { *(float4*)(row + d) = make_float4(x0, x1, x2, x3); });
        if (at.kg == 0) a.ws_ml[slot * 16 + at.c] = make_float2(at.m, l);
      }
    }
    if (left <= 0) return;
    first = 0;
    if (++r == heads) {  // on to the next sequence that has keys
      r = 0;
      do {
        ctx = __builtin_amdgcn_readfirstlane(context_of(a, ++b));
      } while (ctx == 0);
      n = (ctx + kTile - 1) / kTile;
    }
  }
}

// Joins what the runs left of each (sequence, query head), a workgroup each: a thread has
// four dims of every parts-th run, kJoinBatch of them asked for at once, and the threads
// of the same dims meet in LDS. Rows without keys come out 0.
constexpr int kJoinThreads = 256, kJoinBatch = 4;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_fp4_join(const Fp4DecodeArgs a, int dims) {
  __shared__ float4 lds_x[kJoinThreads];
  __shared__ float lds_sum[kJoinThreads];
  const int b = (int)blockIdx.y, h = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63;
  const int hk = h / a.G, g = h - hk * a.G, qt = g >> 4, heads = a.Hk * a.q_tiles, r = hk * a.q_tiles + qt;
  const int at = a.ws_cum[b], n = a.ws_cum[b + 1] - at;
  const int64_t total = (int64_t)a.ws_cum[a.B] * heads;
  T* row = out_row<T>(a, b, h);
  const int quads = dims / 4, parts = kJoinThreads / quads, part = tid / quads, d = (tid - part * quads) * 4;
  if (n == 0) {
    if (part == 0) store4(a, row, d, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  const int64_t p0 = (int64_t)at * heads + (int64_t)r * n, p1 = p0 + n;
  const Runs runs(total, a.waves);
  const int w0 = runs.of(p0), w1 = runs.of(p1 - 1);
  if (w0 == w1) return;
  const int rows = min(a.G, 16);
  const auto slot_of = [&](int w) { return 2 * (int64_t)w + (w == w0); };
  float m = kNoMax, sum = 0.f;
  for (int w = w0 + lane; w <= w1; w += 64) m = fmaxf(m, a.ws_ml[slot_of(w) * 16 + (g & 15)].x);
  m = wave_max(m);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (part < parts) {
    for (int w = w0 + part; w <= w1; w += kJoinBatch * parts) {
      float2 ml[kJoinBatch];
      float4 y[kJoinBatch];
#pragma unroll
      for (int i = 0; i < kJoinBatch; ++i) {
        const int64_t slot = slot_of(min(w + i * parts, w1));
        ml[i] = a.ws_ml[slot * 16 + (g & 15)];
        y[i] = *(const float4*)(a.ws_acc + (slot * rows + (g & 15)) * dims + d);
      }
#pragma unroll
      for (int i = 0; i < kJoinBatch; ++i)
        if (w + i * parts <= w1) {
          const float f = fast_exp2((ml[i].x - m) * a.scale_log2);
          sum += f * ml[i].y;
          x.x += f * y[i].x, x.y += f * y[i].y, x.z += f * y[i].z, x.w += f * y[i].w;
        }
    }
  }
  lds_x[tid] = x;
  lds_sum[tid] = sum;
  __syncthreads();
  if (part != 0) return;
  for (int p = 1; p < parts; ++p) {
    const float4 y = lds_x[p * quads + tid];
    sum += lds_sum[p * quads + tid];
    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
  }
  const float inv = inverse(sum);
  store4(a, row, d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
}

template <typename T, int NG, bool ANY>
hipError_t launch_ng(Fp4DecodeArgs a, hipStream_t stream) {
  void* args[] = {&a, nullptr};
  if (a.one_launch) {
    const size_t lds = (size_t)a.waves * (a.G < 16 ? a.G : 16) * (NG * 32 + 4) * 4;
    return hipLaunchKernel(reinterpret_cast<const void*>(&paged_fp4_one<T, NG, ANY>),
                           dim3((unsigned)(a.B * a.Hk * a.q_tiles)), dim3(a.waves * 64), args, lds, stream);
  }
  hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&paged_fp4_split<T, NG, ANY>),
                                 dim3((unsigned)(a.waves / 4)), dim3(256), args, 0, stream);
  if (e != hipSuccess) return e;
  int dims = NG * 32;
  args[1] = &dims;
  return hipLaunchKernel(reinterpret_cast<const void*>(&paged_fp4_join<T>), dim3(a.Hk * a.G, a.B),
                         dim3(kJoinThreads), args, 0, stream);
}

template <typename T, int NG>
hipError_t launch_any(const Fp4DecodeArgs& a, hipStream_t stream) {
  return a.S % 16 == 0 ? launch_ng<T, NG, false>(a, stream) : launch_ng<T, NG, true>(a, stream);
}

template <typename T>
hipError_t launch_paged_fp4(const Fp4DecodeArgs& a, hipStream_t stream) {
  switch (fp4_groups(a.D)) {
    case 1: return launch_any<T, 1>(a, stream);
    case 2: return launch_any<T, 2>(a, stream);
    case 3: return launch_any<T, 3>(a, stream);
    case 4: return launch_any<T, 4>(a, stream);
    case 5: return launch_any<T, 5>(a, stream);
    case 6: return launch_any<T, 6>(a, stream);
    case 7: return launch_any<T, 7>(a, stream);
    case 8: return launch_any<T, 8>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

}  // namespace mgi
