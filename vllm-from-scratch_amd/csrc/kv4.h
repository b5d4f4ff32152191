// The 4-bit KV cache: E2M1 codes with one E8M0 scale per 32 dims of a token's head row (the OCP
// microscaling format, which this chip converts in one instruction per two values).
//
//   value = code value * 2^(scale byte - 127), code values 0 .5 1 1.5 2 3 4 6 and their negatives;
//   the scale is the smallest power of two with max|x| <= 6 * 2^e, e in [-120, 125]; a block that
//   holds a NaN or an infinity has scale byte 255 and reads as NaN.
//
// A cache tensor is bytes [blocks, kv_heads, block_size / 16, 17 D / 2]: one record per block, head
// and tile of 16 tokens, 8 D bytes of codes and behind them D / 2 scale bytes.  A record is laid
// out as the 16x16x32 matrix instruction wants it (lane l = 16 g + c, g in 0..3), so that a wave
// reads a tile with one load per lane and no exchange between lanes:
//   K  codes [16 tokens][D / 2] (even dim in the low nibble): lane (g, c) takes the D / 8 bytes of
//      token c's dims [g D/4, (g+1) D/4); dword s of them is its part of contraction step s.
//      scales [16 tokens][D / 32]
//   V  codes [4 g][16 c][D / 32 blocks][4 j]: the byte holds dims 32 b + 2 c and 32 b + 2 c + 1 of
//      token 4 g + j: lane (g, c) takes D / 8 consecutive bytes, four tokens of two dims per block.
//      scales [4 g][D / 32][4 j]
// Two tiles make a step of 32 tokens whose contraction index (g, j) is token 4 g + j of the first
// tile for j < 4 and 4 g + j - 4 of the second: the order in which a score tile K Q^T leaves the
// matrix unit, so that weights go back in without moving between lanes.
#pragma once

#include "common.h"

namespace mi355 {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kKv4Tile = 16;          // tokens per record
constexpr int kKv4MaxContext = 1 << 29;   // positions are ints, and a step looks past its end
constexpr int kKv4Step = 32;          // tokens per contraction step: two records
constexpr int kKv4MinExp = -120, kKv4MaxExp = 125;
constexpr float kKv4Floor = -3e38f;   // a running maximum no score has raised yet
// Powers of two a score may pass the running maximum by before it is raised.  Weights are made as much smaller, 2^-8 at the
// maximum: they stay at 1 or below, and values up to the largest that the format holds below the largest float.
constexpr float kKv4Raise = 8.f;

static inline bool kv4_dtype_ok(int dtype) { return dtype == MI355_F32 || dtype == MI355_BF16 || dtype == MI355_F16; }
// A launch has fewer than 2^32 threads.
static inline bool kv4_grid_ok(int64_t workgroups, int threads) { return workgroups <= (int64_t)(UINT32_MAX / (uint32_t)threads); }
static inline bool kv4_head_dim_ok(int D) { return D == 32 || D == 64 || D == 128 || D == 256; }

// Geometry shared by every kernel over the cache; strides in bytes.
struct Kv4Cache {
  char* k;
  char* v;
  int64_t s_blk, s_head;
  int num_blocks, tpb;       // blocks in the pool, tiles per block
  uint32_t tpb_mul;          // tile / tpb = tile * tpb_mul >> tpb_shift for tile < 2^31
  int tpb_shift;
};
static inline Kv4Cache kv4_cache(const void* k, const void* v, int64_t s_blk, int64_t s_head, int num_blocks, int tpb) {
  int up = 0;
  while ((1ll << up) < tpb) ++up;
  const uint32_t mul = (uint32_t)(((1ull << (31 + up)) + tpb - 1) / tpb);   // ceil(2^(31+up) / tpb) <= 2^31 + ...: fits
  return Kv4Cache{static_cast<char*>(const_cast<void*>(k)), static_cast<char*>(const_cast<void*>(v)), s_blk, s_head,
                  num_blocks, tpb, mul, 31 + up};
}
// Whether `out` (contiguous) and the span of T rows from x share bytes.
static inline bool kv4_overlaps(const char* out, int64_t out_bytes, const char* x, int64_t stride, int64_t width, int T) {
  return out < x + ((int64_t)(T - 1) * stride + width) && x < out + out_bytes;
}
// An output of attention may be the query rows themselves (a workgroup reads its own before it writes them), but share no
// bytes with them otherwise.
static inline bool kv4_out_ok(const void* out, const void* q, int64_t q_stride, int64_t row, int T, int dtype) {
  const int64_t eb = dtype == MI355_F32 ? 4 : 2;
  return (out == q && (q_stride == row || T == 1)) ||
         !kv4_overlaps(static_cast<const char*>(out), T * row * eb, static_cast<const char*>(q), q_stride * eb, row * eb, T);
}
// Checks what every entry point over the cache asks of it; 0 or the recorded error.
int kv4_check_cache(const char* what, const void* k_cache, const void* v_cache, int Hkv, int D, int block_size,
                    int num_blocks, int64_t s_blk, int64_t s_head);

__device__ __forceinline__ constexpr int kv4_tile_bytes(int D) { return 17 * D / 2; }

// Where tile `tile` of a sequence lies: the table entry that names its block, and its place in the block.
struct Kv4Place {
  int id, sub;
};
__device__ __forceinline__ Kv4Place kv4_place(const Kv4Cache& c, const int32_t* table, int tile) {
  const int blk = (int)(((uint64_t)(uint32_t)tile * c.tpb_mul) >> c.tpb_shift);
  // (constant memory for this launch, and the index is uniform: a scalar load, which vector loads in flight need not wait for)
  typedef const __attribute__((address_space(4))) int32_t* ctable;
  return Kv4Place{((ctable)table)[blk], tile - blk * c.tpb};
}
// Byte offset of its record within a head's part of the pool.
__device__ __forceinline__ int64_t kv4_record(const Kv4Cache& c, Kv4Place at, int tile_bytes) {
  const int id = at.id < 0 ? 0 : (at.id >= c.num_blocks ? c.num_blocks - 1 : at.id);
  return (int64_t)((uint64_t)(uint32_t)id * (uint64_t)c.s_blk) + (int64_t)at.sub * tile_bytes;   // (a block may pass 2^31 bytes)
}

// E8M0 byte j of a dword -> the scale operand of the conversion instructions, which read the exponent
// field of a float and nothing else (255 is answered with NaN): one shift, whatever lands in the sign
// and the fraction.
__device__ __forceinline__ float kv4_scale(uint32_t w, int j) {
  return u2f(j == 3 ? w >> 1 : w << (23 - 8 * j));
}

// Byte J of `w` -> (low nibble, high nibble) as two bf16, times the scale: exact for every scale that the append writes
// (bytes 253 and 254 lead beyond the largest bf16: infinities).
template <int J>
__device__ __forceinline__ uint32_t kv4_to_bf16(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, J));
}

union Bf16Frag {
  uint32_t w[4];
  bf16x8_t v;
};

// One contraction step of a K tile: eight dims of one token.
__device__ __forceinline__ bf16x8_t kv4_k_frag(uint32_t w, float scale) {
  Bf16Frag f;
  f.w[0] = kv4_to_bf16<0>(w, scale);
  f.w[1] = kv4_to_bf16<1>(w, scale);
  f.w[2] = kv4_to_bf16<2>(w, scale);
  f.w[3] = kv4_to_bf16<3>(w, scale);
  return f.v;
}

// One block of 32 dims of a V step: dwords w0 / w1 and scale dwords s0 / s1 of its two tiles ->
// the operands of the even and of the odd dims (row c = dim 32 b + 2 c (+ 1), contraction = token).
__device__ __forceinline__ void kv4_v_frags(uint32_t w0, uint32_t w1, uint32_t s0, uint32_t s1, bf16x8_t& even,
                                            bf16x8_t& odd) {
  uint32_t r[8];
  r[0] = kv4_to_bf16<0>(w0, kv4_scale(s0, 0));
  r[1] = kv4_to_bf16<1>(w0, kv4_scale(s0, 1));
  r[2] = kv4_to_bf16<2>(w0, kv4_scale(s0, 2));
  r[3] = kv4_to_bf16<3>(w0, kv4_scale(s0, 3));
  r[4] = kv4_to_bf16<0>(w1, kv4_scale(s1, 0));
  r[5] = kv4_to_bf16<1>(w1, kv4_scale(s1, 1));
  r[6] = kv4_to_bf16<2>(w1, kv4_scale(s1, 2));
  r[7] = kv4_to_bf16<3>(w1, kv4_scale(s1, 3));
  Bf16Frag e, o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e.w[i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x05040100u);
    o.w[i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x07060302u);
  }
  even = e.v;
  odd = o.v;
}

__device__ __forceinline__ f32x4 mfma_bf16(bf16x8_t a, bf16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// N = 1, 2, 3 bf16 pieces of eight floats whose sum is the float to 8, 16, 24 bits: what makes the
// bf16 matrix instruction exact for bf16, fp16 and fp32 operands against codes that bf16 holds
// exactly.  (An fp32 value above bf16's largest, 3.39e38, counts as an infinity.)
template <int N>
__device__ __forceinline__ void bf16_pieces(const float (&x)[8], bf16x8_t (&out)[N]) {
  float rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const __bf16 h = (__bf16)rest[e];
      out[n][e] = h;
      if (n + 1 < N) rest[e] -= (float)h;
    }
  }
}

// The same of eight softmax weights, with one instruction for what a rounding leaves of a weight instead of two: the dot
// product of the rounded pair with (-1, 0) or (0, -1), added to the weight (exact, as the difference is).  The two pairs of
// constants stay in registers: as an inline constant of this instruction -1 is not the pair that the compiler takes it for.
template <int N>
__device__ __forceinline__ void weight_pieces(const float (&x)[8], bf16x8_t (&out)[N]) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  uint32_t first = 0x0000bf80u, second = 0xbf800000u;
  asm("" : "+s"(first), "+s"(second));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float a = x[e], b = x[e + 1];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const bf16x2_t h = {(__bf16)a, (__bf16)b};
      out[n][e] = h[0];
      out[n][e + 1] = h[1];
      if (n + 1 < N) {
        a = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2_t, first), a, false);
        b = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2_t, second), b, false);
      }
    }
  }
}

// Pieces of a query (all of its bits) and of a softmax weight.  A weight takes two at least: in one piece the rows of bf16
// queries move by as much as their own rounding does (1.7e-3 of a row from the exact one, 2.3e-3 in one piece); in two
// they move by 2^-17.  The second piece costs 4 x 2048 rows behind 2048, 32/8 heads of 128, 560 us for 417, 8 chunks behind
// 900 10.3 for 9.7, and decode, which memory bounds, under 1 %.
template <class Tag>
struct Kv4Pieces;
template <>
struct Kv4Pieces<BF16> { static constexpr int n = 1, weights = 2; };
template <>
struct Kv4Pieces<F16> { static constexpr int n = 2, weights = 2; };
template <>
struct Kv4Pieces<F32> { static constexpr int n = 3, weights = 3; };

// Eight consecutive elements of a row (16-byte aligned) as floats, and back with one rounding.
template <class Tag>
__device__ __forceinline__ void load8(const char* p, float (&x)[8]) {
  if constexpr (Tag::kBytes == 4) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    Tag::unpack(*reinterpret_cast<const u32x4*>(p), x);
  }
}
template <class Tag>
__device__ __forceinline__ void store8(char* p, const float (&x)[8]) {
  if constexpr (Tag::kBytes == 4) {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(p + 16) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<u32x4*>(p) = Tag::pack(x);
  }
}

// A tile's K and V registers of one kv head.
template <int D>
struct Kv4TileRegs {
  uint32_t k[D / 32], v[D / 32], vs[D / 32];
  uint32_t ks;   // the dword that holds the scale byte(s) of the lane's dims [g D/4, +D/4)
};

typedef const __attribute__((address_space(1))) char* gptr;   // (an address that passes through asm has to say that it is global)

// NT: rows that one workgroup reads once bypass the caches' retention.
template <bool NT, int W>
__device__ __forceinline__ void load_words(gptr p, uint32_t (&w)[W]) {
  auto get = [](auto* q) { return NT ? __builtin_nontemporal_load(q) : *q; };
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef const __attribute__((address_space(1))) uint32_t* p1;
  typedef const __attribute__((address_space(1))) u32x2* p2;
  typedef const __attribute__((address_space(1))) u32x4* p4;
  if constexpr (W == 1) {
    w[0] = get((p1)p);
  } else if constexpr (W == 2) {
    const u32x2 a = get((p2)p);
    w[0] = a[0], w[1] = a[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 a = get((p4)(p + 4 * i));
      w[i] = a[0], w[i + 1] = a[1], w[i + 2] = a[2], w[i + 3] = a[3];
    }
  }
}

// Where a lane finds its parts of a record (unsigned, so that a load is a uniform base and a 32-bit
// lane offset), and by how much its K scale byte has to turn within its dword to land in the
// exponent field.
template <int D>
struct Kv4Lane {
  uint32_t k, ks, v, vs, turn;
  __device__ __forceinline__ explicit Kv4Lane(int lane) {
    const uint32_t g = (uint32_t)lane >> 4, c = (uint32_t)lane & 15;
    k = c * (D / 2) + g * (D / 8);
    v = (uint32_t)lane * (D / 8);
    vs = 8 * D + g * (D / 8);
    const uint32_t at = c * (D / 32) + (g * (D / 4)) / 32;   // the lane's (first) scale byte
    ks = 8 * D + (at & ~3u);
    turn = (9 + 8 * (at & 3)) & 31;
  }
};
// A uniform address kept in scalar registers: left alone, the compiler adds the loop's invariant part
// of an address to the lane offsets and pays a 64-bit vector addition per load.
__device__ __forceinline__ gptr scalar_base(const char* p) {
  gptr g = (gptr)p;
  asm("" : "+s"(g));
  return g;
}
// The lane's 32-bit offset, as a value the compiler cannot widen outside the loop (the widening has to
// stand next to the load for the load to take a scalar base and a 32-bit offset).
__device__ __forceinline__ uint32_t lane_offset(uint32_t& o) {
  asm volatile("" : "+v"(o));
  return o;
}
template <int D, bool NT>
__device__ __forceinline__ void kv4_load_k(gptr rec, Kv4Lane<D>& at, Kv4TileRegs<D>& t) {
  load_words<NT>(rec + lane_offset(at.k), t.k);
  uint32_t s[1];
  load_words<NT>(rec + lane_offset(at.ks), s);
  t.ks = s[0];
}
template <int D, bool NT>
__device__ __forceinline__ void kv4_load_v(gptr rec, Kv4Lane<D>& at, Kv4TileRegs<D>& t) {
  load_words<NT>(rec + lane_offset(at.v), t.v);
  load_words<NT>(rec + lane_offset(at.vs), t.vs);
}
// The scale of contraction step s (of D / 32): a lane's dims span one scale block, two at D = 256.
template <int D>
__device__ __forceinline__ float kv4_k_scale(const Kv4TileRegs<D>& t, const Kv4Lane<D>& at, int s) {
  const uint32_t turn = D == 256 && s >= 4 ? (at.turn + 8) & 31 : at.turn;
  return u2f(__builtin_amdgcn_alignbit(t.ks, t.ks, turn));
}

// The softmax weight of a score against a running maximum.  (The difference first: it is exact near the maximum however
// large the two are, which the difference of their products with the scale is not -- 2^31 would be off by 2^7.)
__device__ __forceinline__ float kv4_weight(float score, float m, float scale2) {
  return fast_exp2(__builtin_fmaf(score - m, scale2, -kKv4Raise));
}
// What sums that belong to maximum `from` are worth under maximum `to`.
__device__ __forceinline__ float kv4_shift(float from, float to, float scale2) { return fast_exp2((from - to) * scale2); }

// Joins a row's `n` split records of D + 4 floats (unnormalised sums, running maximum of the raw scores, sum of weights)
// and stores the row.  A thread owns eight dims and every SL-th split, SL * D / 8 threads a row; with
// SL > 1 the row is the whole workgroup's (256 threads) and its threads of the same dims meet in LDS.
// The records of a row lie a memory latency apart when one thread walks them (32 splits of 128 dims:
// 25 us), but a workgroup per row is too much for thousands of rows of a few splits (12 prompts of 64
// dims in two splits: 162 us in all, 48 unsplit): kv4_split_lanes picks by the number of splits.
constexpr int kKv4WalkedSplits = 8;
template <int D>
constexpr int kv4_split_lanes(bool walked) { return walked ? 1 : 256 / (D / 8); }
template <class Tag, int D, int SL>
__device__ inline void kv4_join_splits(char* out, const float* ws, int n, float scale2) {
  constexpr int P = D / 8;
  __shared__ float s_m[SL][P], s_l[SL][P], s_o[SL][P][9];   // (9: neighbouring threads on neighbouring banks)
  const int piece = threadIdx.x % P, sl = SL == 1 ? 0 : threadIdx.x / P;
  float M = kKv4Floor, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto join = [&](float ms, float ls, const float (&x)[8]) {
    const float Mn = fmaxf(M, ms), fo = kv4_shift(M, Mn, scale2), fn = kv4_shift(ms, Mn, scale2);
    M = Mn;
    L = __builtin_fmaf(ls, fn, L * fo);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf(x[e], fn, o[e] * fo);
  };
#pragma unroll 4
  for (int s = sl; s < n; s += SL) {
    const float* rec = ws + (int64_t)s * (D + 4);
    float x[8];
    load8<F32>(reinterpret_cast<const char*>(rec + piece * 8), x);
    join(rec[D], rec[D + 1], x);
  }
  for (int half = SL / 2; half > 0; half /= 2) {
    if (sl >= half && sl < 2 * half) {
      s_m[sl][piece] = M;
      s_l[sl][piece] = L;
#pragma unroll
      for (int e = 0; e < 8; ++e) s_o[sl][piece][e] = o[e];
    }
    __syncthreads();
    if (sl < half) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s_o[sl + half][piece][e];
      join(s_m[sl + half][piece], s_l[sl + half][piece], x);
    }
  }
  if (sl != 0) return;
  const float inv = n > 0 ? 1.f / L : 0.f;   // no token at all: zeros
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = n > 0 ? o[e] * inv : 0.f;
  store8<Tag>(out + piece * 8 * Tag::kBytes, o);
}

}  // namespace mi355
