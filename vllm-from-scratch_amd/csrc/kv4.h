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
constexpr int kKv4Step = 32;          // tokens per contraction step: two records
constexpr int kKv4MinExp = -120, kKv4MaxExp = 125;
constexpr float kKv4Floor = -3e38f;   // a running maximum no score has raised yet
constexpr float kKv4Raise = 8.f;      // powers of two a score may pass the running maximum by before it is raised

static inline bool kv4_dtype_ok(int dtype) { return dtype == MI355_F32 || dtype == MI355_BF16 || dtype == MI355_F16; }
static inline bool kv4_head_dim_ok(int D) { return D == 32 || D == 64 || D == 128 || D == 256; }

// Geometry shared by every kernel over the cache; strides in bytes.
struct Kv4Cache {
  char* k;
  char* v;
  int64_t s_blk, s_head;
  int num_blocks, tpb;   // blocks in the pool, tiles per block
};

// Checks what every entry point over the cache asks of it; 0 or the recorded error.
int kv4_check_cache(const char* what, const void* k_cache, const void* v_cache, int Hkv, int D, int block_size,
                    int num_blocks, int64_t s_blk, int64_t s_head);

__device__ __forceinline__ constexpr int kv4_tile_bytes(int D) { return 17 * D / 2; }

// E8M0 byte j of a dword -> the float 2^(byte - 127) that the conversion instructions take
// (255 becomes the pattern they answer with NaN).
__device__ __forceinline__ float kv4_scale(uint32_t w, int j) { return u2f(((w >> (8 * j)) & 0xffu) << 23); }

// Byte J of `w` -> (low nibble, high nibble) as two bf16, times the scale: exact.
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
// exactly.  (A value beyond bf16's range never occurs: fp32 and bf16 share the exponent.)
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

template <class Tag>
struct Kv4Pieces;
template <>
struct Kv4Pieces<BF16> { static constexpr int n = 1; };
template <>
struct Kv4Pieces<F16> { static constexpr int n = 2; };
template <>
struct Kv4Pieces<F32> { static constexpr int n = 3; };

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
  uint32_t ks;   // scale bytes of the lane's dims [g D/4, +D/4)
};

template <int W>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[W]) {
  if constexpr (W == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (W == 2) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    w[0] = a.x, w[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(p + 4 * i);
      w[i] = a[0], w[i + 1] = a[1], w[i + 2] = a[2], w[i + 3] = a[3];
    }
  }
}

template <int D>
__device__ __forceinline__ void kv4_load_k(const char* rec, int lane, Kv4TileRegs<D>& t) {
  const int g = lane >> 4, c = lane & 15;
  load_words(rec + c * (D / 2) + g * (D / 8), t.k);
  const char* s = rec + 8 * D + c * (D / 32);
  if constexpr (D == 32) t.ks = *reinterpret_cast<const uint8_t*>(s);
  else if constexpr (D == 64) t.ks = *reinterpret_cast<const uint8_t*>(s + (g >> 1));
  else if constexpr (D == 128) t.ks = *reinterpret_cast<const uint8_t*>(s + g);
  else t.ks = *reinterpret_cast<const uint16_t*>(s + 2 * g);
}
template <int D>
__device__ __forceinline__ void kv4_load_v(const char* rec, int lane, Kv4TileRegs<D>& t) {
  load_words(rec + lane * (D / 8), t.v);
  load_words(rec + 8 * D + (lane >> 4) * (D / 8), t.vs);
}

}  // namespace mi355
