// Rows on their way into (and out of) the 4-bit KV cache:
//
//   rope_angles_kernel     cos / sin rows of a step's positions from a frequency per pair
//   kv4_append_kernel      rotation of query, key (and of nothing else) rows, E2M1 / E8M0 rounding of
//                          key and value rows, scatter into the cache's records by slot id
//   kv4_read_kernel        cached rows by slot id as values
//
// All are byte movers; every row is read once and written once.  8192 tokens with 32/8 heads of 128 in bf16: append 181 MB in
// 37.6 us, read-back 42 MB in 12.0 (a 1 GiB copy: 5.16 TB/s).
#include "kv4.h"

namespace mi355 {

int kv4_check_cache(const char* what, const void* k_cache, const void* v_cache, int Hkv, int D, int block_size,
                    int num_blocks, int64_t s_blk, int64_t s_head) {
  if (!k_cache || !v_cache) return fail(MI355_EINVAL, "%s: null pointer argument", what);
  if (!kv4_head_dim_ok(D)) return fail(MI355_EUNSUPPORTED, "%s: head_dim %d (the 4-bit cache holds 32, 64, 128 or 256)", what, D);
  if (Hkv <= 0 || num_blocks <= 0) return fail(MI355_EINVAL, "%s: bad shape (Hkv=%d num_blocks=%d)", what, Hkv, num_blocks);
  if (block_size <= 0 || block_size % kKv4Tile)
    return fail(MI355_EUNSUPPORTED, "%s: block_size %d (the 4-bit cache keeps tiles of %d tokens)", what, block_size, kKv4Tile);
  const int64_t head = (int64_t)(block_size / kKv4Tile) * (17 * D / 2);
  if (s_head % 16 || s_blk % 16 || (Hkv > 1 && s_head < head) || (num_blocks > 1 && s_blk < head) || s_head < 0 || s_blk < 0 ||
      (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15))
    return fail(MI355_EINVAL, "%s: cache records must be 16-byte aligned and a head's tiles contiguous", what);
  return 0;
}

namespace {

// ---------------------------------------------------------------------------
// angles
// ---------------------------------------------------------------------------
// a = position * frequency is formed in double: at position 2^24 a float's last bit is a whole
// radian.  Reduction to [-pi/4, pi/4] with pi/2 in two parts, then the Taylor polynomials: the first
// term left out is below 7e-12, far under the float the result is rounded to.  The rounding of
// a * 2 / pi moves the quotient by 2^-13 at 2^40 and by whole turns beyond 2^53, so far angles are
// reduced a second time.  (Beyond 2^63, where no 64-bit position leads at a frequency of 1: NaN.)
__device__ __forceinline__ void sincos_reduced(double a, double& s, double& c) {
  constexpr double kTurns = 0.63661977236758134308;                            // 2 / pi
  constexpr double kHi = 1.57079632679489655800e+00, kLo = 6.12323399573676603587e-17;
  const double n = __builtin_rint(a * kTurns);
  double r = __builtin_fma(-n, kHi, a);
  r = __builtin_fma(-n, kLo, r);
  long long quarter = (long long)n;
  if (!(__builtin_fabs(a) < 0x1p40)) {
    const double m = __builtin_rint(r * kTurns);
    r = __builtin_fma(-m, kHi, r);
    r = __builtin_fma(-m, kLo, r);
    quarter += (long long)m;
    if (!(__builtin_fabs(a) <= 0x1p63)) r = __builtin_nan("");
  }
  const double z = r * r;
  double ps = -1.0 / 39916800.0;
  ps = __builtin_fma(ps, z, 1.0 / 362880.0);
  ps = __builtin_fma(ps, z, -1.0 / 5040.0);
  ps = __builtin_fma(ps, z, 1.0 / 120.0);
  ps = __builtin_fma(ps, z, -1.0 / 6.0);
  const double sr = __builtin_fma(ps * z, r, r);
  double pc = 1.0 / 479001600.0;
  pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
  pc = __builtin_fma(pc, z, 1.0 / 40320.0);
  pc = __builtin_fma(pc, z, -1.0 / 720.0);
  pc = __builtin_fma(pc, z, 1.0 / 24.0);
  pc = __builtin_fma(pc, z, -0.5);
  const double cr = __builtin_fma(pc, z, 1.0);
  const int q = (int)quarter & 3;
  const double sv = (q & 1) ? cr : sr, cv = (q & 1) ? sr : cr;
  s = (q & 2) ? -sv : sv;
  c = (q == 1 || q == 2) ? -cv : cv;
}

__global__ void __launch_bounds__(256)
rope_angles_kernel(float* cos_out, float* sin_out, const int64_t* positions, const double* inv_freq, double factor,
                   int64_t total, int half) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= total) return;
  const int64_t t = idx / half;
  const int i = (int)(idx - t * half);
  double s, c;
  sincos_reduced((double)positions[t] * inv_freq[i], s, c);
  cos_out[idx] = (float)(c * factor);
  sin_out[idx] = (float)(s * factor);
}

// ---------------------------------------------------------------------------
// rotation + append
// ---------------------------------------------------------------------------
struct AppendParams4 {
  const char* q;
  const char* k;
  const char* v;
  const float* cos;   // [T, R / 2], null: no rotation
  const float* sin;
  const int64_t* slots;   // null: rotate the query heads only
  char* q_out;            // [T, Hq, D]
  Kv4Cache cache;
  int64_t q_stride_tok, k_stride_tok, v_stride_tok;   // elements
  int64_t rows, num_slots;                            // rows = token groups * heads
  int T, Hq, Hkv, heads /* Hq + 2 Hkv, or Hq */, R, bs_shift;
};

// A double as a float that keeps on which side of every float it lies (round to odd): the 4-bit
// rounding that follows then decides as it would on the double itself.
__device__ __forceinline__ float round_to_odd(double d) {
  const float f = (float)d;
  uint32_t b = f2u(f);
  const double back = (double)f;
  if (back != d) {
    b -= __builtin_fabs(back) > __builtin_fabs(d) ? 1u : 0u;
    b |= 1u;
  }
  return u2f(b);
}

// Row -> eight codes per thread and the scale of the 32 dims that four neighbouring threads hold.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& scale_byte) {
  uint32_t top = 0;   // |x| as integers: order of magnitudes, NaN and infinity on top
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = f2u(x[e]) & 0x7fffffffu;
    top = u > top ? u : top;
  }
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false);
  top = o > top ? o : top;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false);
  top = o > top ? o : top;
  int e = (int)(top >> 23) - 129 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0);
  e = e < kKv4MinExp ? kKv4MinExp : (e > kKv4MaxExp ? kKv4MaxExp : e);
  const bool bad = top >= 0x7f800000u;
  scale_byte = bad ? 255u : (uint32_t)(e + 127);
  const float sc = u2f((uint32_t)(e + 127) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], sc, 3);
  return w;
}

// Where a slot's record of one head begins, and the token's place in it.
template <int D>
__device__ __forceinline__ int64_t slot_record(const Kv4Cache& c, int64_t slot, int bs_shift, int h, int& r) {
  const int64_t blk = bs_shift >= 0 ? (slot >> bs_shift) : slot / (c.tpb * kKv4Tile);
  const int in = (int)(slot - blk * c.tpb * kKv4Tile);
  r = in % kKv4Tile;
  return blk * c.s_blk + (int64_t)h * c.s_head + (int64_t)(in / kKv4Tile) * kv4_tile_bytes(D);
}
// Whether two tokens' codes are neighbouring bytes of a value record, in order.
__device__ __forceinline__ bool one_pair(int64_t a, int64_t b) { return a % 2 == 0 && b == a + 1; }

// Thread = eight dims of one head row of N neighbouring tokens; D / 8 threads hold a row, rows are
// (token group, head slot) with the query heads first, the key heads next and the value heads last.
template <class Tag, int D, bool INTER, int N>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendParams4 p) {
  constexpr int EB = Tag::kBytes, P = D / 8, NB = D / 32, RPB = 256 / P;
  const int piece = threadIdx.x % P;
  const int64_t row0 = (int64_t)blockIdx.x * RPB;
  const int64_t g0 = row0 / p.heads;                                   // uniform
  const int local = (int)(row0 - g0 * p.heads) + (int)threadIdx.x / P;
  const int64_t t0 = (g0 + local / p.heads) * N;
  const int hs = local % p.heads;
  if (row0 + threadIdx.x / P >= p.rows) return;

  const bool is_q = hs < p.Hq, is_k = !is_q && hs < p.Hq + p.Hkv;
  const int h = is_q ? hs : (is_k ? hs - p.Hq : hs - p.Hq - p.Hkv);
  const int64_t stride = (is_q ? p.q_stride_tok : is_k ? p.k_stride_tok : p.v_stride_tok) * EB;
  const char* const src = (is_q ? p.q : is_k ? p.k : p.v) + t0 * stride + h * D * EB;
  int64_t slot[N];
  bool live[N];   // (the four threads of a block of dims agree)
  float x[N][8];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const bool in = t0 + n < p.T;
    slot[n] = !is_q && in ? p.slots[t0 + n] : -1;
    live[n] = in && (is_q || (slot[n] >= 0 && slot[n] < p.num_slots));
    load8<Tag>(src + (in ? n : 0) * stride + piece * 8 * EB, x[n]);
  }

  if ((is_q || is_k) && p.cos && piece * 8 < p.R) {
    const int half = p.R / 2;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int m = t0 + n < p.T ? n : 0;
      float y[8], c[8], s[8];
      const float* cr = p.cos + (t0 + m) * half;
      const float* sr = p.sin + (t0 + m) * half;
      if constexpr (INTER) {   // pairs (2 i, 2 i + 1): the partner is the neighbour
        const f32x4 c4 = *reinterpret_cast<const f32x4*>(cr + piece * 4), s4 = *reinterpret_cast<const f32x4*>(sr + piece * 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = x[n][e ^ 1];
          c[e] = c4[e / 2];
          s[e] = (e & 1) ? s4[e / 2] : -s4[e / 2];
        }
      } else {                 // pairs (i, i + R / 2): the partner row piece is read again (it is in the cache)
        const bool low = piece * 8 < half;
        const int i = low ? piece * 8 : piece * 8 - half;
        load8<Tag>(src + m * stride + (low ? piece * 8 + half : i) * EB, y);
        const f32x4 ca = *reinterpret_cast<const f32x4*>(cr + i), cb = *reinterpret_cast<const f32x4*>(cr + i + 4);
        const f32x4 sa = *reinterpret_cast<const f32x4*>(sr + i), sb = *reinterpret_cast<const f32x4*>(sr + i + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[e] = ca[e];
          c[4 + e] = cb[e];
          s[e] = low ? -sa[e] : sa[e];
          s[4 + e] = low ? -sb[e] : sb[e];
        }
      }
      if (is_q) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[n][e] = __builtin_fmaf(x[n][e], c[e], y[e] * s[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[n][e] = round_to_odd(__builtin_fma((double)x[n][e], (double)c[e], (double)y[e] * (double)s[e]));
      }
    }
  }
  if (is_q) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (live[n]) store8<Tag>(p.q_out + (((t0 + n) * p.Hq + h) * D + piece * 8) * EB, x[n]);
    return;
  }
  uint32_t w[N], sb[N];
#pragma unroll
  for (int n = 0; n < N; ++n) w[n] = quantise8(x[n], sb[n]);
  char* const pool = is_k ? p.cache.k : p.cache.v;
  if constexpr (N == 2) {
    if (!is_k && live[0] && live[1] && one_pair(slot[0], slot[1])) {   // (prompts)
      int r;
      char* rec = pool + slot_record<D>(p.cache, slot[0], p.bs_shift, h, r) + r % 4;
      const int b = piece / 4, c0 = (piece % 4) * 4;
      const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), hi = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint16_t*>(rec + ((r / 4 * 16 + c0 + i) * NB + b) * 4) = (uint16_t)((i < 2 ? lo : hi) >> (i % 2 * 16));
      if (piece % 4 == 0) *reinterpret_cast<uint16_t*>(rec + 8 * D + (r / 4 * NB + b) * 4) = (uint16_t)(sb[0] | sb[1] << 8);
      return;
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!live[n]) continue;
    int r;
    char* rec = pool + slot_record<D>(p.cache, slot[n], p.bs_shift, h, r);
    if (is_k) {
      *reinterpret_cast<uint32_t*>(rec + r * (D / 2) + piece * 4) = w[n];
      if (piece % 4 == 0) rec[8 * D + r * NB + piece / 4] = (char)sb[n];
    } else {
      const int b = piece / 4, c0 = (piece % 4) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) rec[((r / 4 * 16 + c0 + i) * NB + b) * 4 + r % 4] = (char)(w[n] >> (8 * i));
      if (piece % 4 == 0) rec[8 * D + (r / 4 * NB + b) * 4 + r % 4] = (char)sb[n];
    }
  }
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
struct ReadParams4 {
  char* k_out;   // [T, Hkv, D]
  char* v_out;
  const int64_t* slots;
  Kv4Cache cache;
  int64_t rows, num_slots;   // rows = token groups * 2 Hkv
  int T, Hkv, bs_shift;
};

template <class Tag, int D, int N>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadParams4 p) {
  constexpr int EB = Tag::kBytes, P = D / 8, NB = D / 32, RPB = 256 / P;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const int piece = threadIdx.x % P, heads = 2 * p.Hkv;
  const int64_t row0 = (int64_t)blockIdx.x * RPB;
  const int64_t g0 = row0 / heads;
  const int local = (int)(row0 - g0 * heads) + (int)threadIdx.x / P;
  const int64_t t0 = (g0 + local / heads) * N;
  const int hs = local % heads;
  if (row0 + threadIdx.x / P >= p.rows) return;
  const bool is_k = hs < p.Hkv;
  const int h = is_k ? hs : hs - p.Hkv, b = piece / 4, c0 = (piece % 4) * 4;
  const uint8_t* const pool = reinterpret_cast<const uint8_t*>(is_k ? p.cache.k : p.cache.v);
  int64_t slot[N];
  bool live[N];
  uint32_t w[N], sb[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    slot[n] = t0 + n < p.T ? p.slots[t0 + n] : -1;
    live[n] = slot[n] >= 0 && slot[n] < p.num_slots;
    w[n] = sb[n] = 0;
  }
  bool done = false;
  if constexpr (N == 2) {
    if (!is_k && live[0] && live[1] && one_pair(slot[0], slot[1])) {
      int r;
      const uint8_t* rec = pool + slot_record<D>(p.cache, slot[0], p.bs_shift, h, r) + r % 4;
      uint32_t d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = *reinterpret_cast<const uint16_t*>(rec + ((r / 4 * 16 + c0 + i) * NB + b) * 4);
      const uint32_t both = *reinterpret_cast<const uint16_t*>(rec + 8 * D + (r / 4 * NB + b) * 4);
      const uint32_t lo = d[0] | d[1] << 16, hi = d[2] | d[3] << 16;
      w[0] = __builtin_amdgcn_perm(hi, lo, 0x06040200u);
      w[1] = __builtin_amdgcn_perm(hi, lo, 0x07050301u);
      sb[0] = both & 0xffu;
      sb[1] = both >> 8;
      done = true;
    }
  }
  if (!done) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!live[n]) continue;
      int r;
      const uint8_t* rec = pool + slot_record<D>(p.cache, slot[n], p.bs_shift, h, r);
      if (is_k) {
        w[n] = *reinterpret_cast<const uint32_t*>(rec + r * (D / 2) + piece * 4);
        sb[n] = rec[8 * D + r * NB + b];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[n] |= (uint32_t)rec[((r / 4 * 16 + c0 + i) * NB + b) * 4 + r % 4] << (8 * i);
        sb[n] = rec[8 * D + (r / 4 * NB + b) * 4 + r % 4];
      }
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (t0 + n >= p.T) continue;
    const float sc = kv4_scale(sb[n], 0);   // (a slot outside the cache: codes 0, values 0)
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[n], sc, 0), bb = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[n], sc, 1);
    const f32x2 cc = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[n], sc, 2), dd = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[n], sc, 3);
    const float x[8] = {a[0], a[1], bb[0], bb[1], cc[0], cc[1], dd[0], dd[1]};
    store8<Tag>((is_k ? p.k_out : p.v_out) + (((t0 + n) * p.Hkv + h) * D + piece * 8) * EB, x);
  }
}

// Two tokens per thread have twice the bytes in flight and store value codes by twos, one token has twice the threads: two pay
// once the chip (2^19 threads at a time) is filled several times over.  us, one / two: rotation + append of 8192 x 48 heads of
// 128 42.7 / 38.7, its read-back 14.0 / 12.5, both for 4096 x 24 heads of 256 36.3 / 32.8; for 1024 x 48 of 128 13.4 / 13.8,
// for 256 x 24 of 64 6.8 / 8.2.  (Four per thread: 41.6 and 12.7.)
bool by_twos(int64_t rows, int D) { return rows * (D / 8) >= 3 << 19; }

template <class Tag, int D, int N>
void launch_append(const AppendParams4& p, bool inter, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div64(p.rows, 256 / (D / 8))), block(256);
  if (inter) hipLaunchKernelGGL((kv4_append_kernel<Tag, D, true, N>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((kv4_append_kernel<Tag, D, false, N>), grid, block, 0, s, p);
}
template <class Tag, int N>
int launch_append(const AppendParams4& p, int D, bool inter, hipStream_t s) {
  switch (D) {
    case 32: launch_append<Tag, 32, N>(p, inter, s); break;
    case 64: launch_append<Tag, 64, N>(p, inter, s); break;
    case 128: launch_append<Tag, 128, N>(p, inter, s); break;
    default: launch_append<Tag, 256, N>(p, inter, s); break;
  }
  return check_launch("kv4_append_kernel");
}
template <class Tag>
int launch_append(AppendParams4& p, int D, bool inter, hipStream_t s) {
  const bool two = by_twos((int64_t)p.T * p.heads, D);
  p.rows = ceil_div64(p.T, two ? 2 : 1) * p.heads;
  return two ? launch_append<Tag, 2>(p, D, inter, s) : launch_append<Tag, 1>(p, D, inter, s);
}
template <class Tag, int D, int N>
void launch_read(const ReadParams4& p, hipStream_t s) {
  hipLaunchKernelGGL((kv4_read_kernel<Tag, D, N>), dim3((unsigned)ceil_div64(p.rows, 256 / (D / 8))), dim3(256), 0, s, p);
}
template <class Tag, int N>
int launch_read(const ReadParams4& p, int D, hipStream_t s) {
  switch (D) {
    case 32: launch_read<Tag, 32, N>(p, s); break;
    case 64: launch_read<Tag, 64, N>(p, s); break;
    case 128: launch_read<Tag, 128, N>(p, s); break;
    default: launch_read<Tag, 256, N>(p, s); break;
  }
  return check_launch("kv4_read_kernel");
}
template <class Tag>
int launch_read(ReadParams4& p, int D, hipStream_t s) {
  const bool two = by_twos((int64_t)p.T * 2 * p.Hkv, D);
  p.rows = ceil_div64(p.T, two ? 2 : 1) * 2 * p.Hkv;
  return two ? launch_read<Tag, 2>(p, D, s) : launch_read<Tag, 1>(p, D, s);
}

// Query (and, with slots, key / value) rows through kv4_append_kernel.
int append_impl(const char* what, AppendParams4& p, int T, int D, int rotary_dim, int interleaved, int dtype,
                hipStream_t s) {
  if (!kv4_dtype_ok(dtype)) return fail(MI355_EINVAL, "%s: dtype %d", what, dtype);
  if (!kv4_head_dim_ok(D)) return fail(MI355_EUNSUPPORTED, "%s: head_dim %d (32, 64, 128 or 256)", what, D);
  if (T < 0 || p.Hq <= 0 || p.Hkv < 0) return fail(MI355_EINVAL, "%s: bad shape (T=%d Hq=%d Hkv=%d)", what, T, p.Hq, p.Hkv);
  if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 16)
    return fail(MI355_EINVAL, "%s: rotary_dim %d must be a multiple of 16 up to head_dim %d", what, rotary_dim, D);
  if (rotary_dim > 0 && (!p.cos || !p.sin)) return fail(MI355_EINVAL, "%s: rotary_dim %d without cos / sin rows", what, rotary_dim);
  const int epl = dtype == MI355_F32 ? 4 : 8;
  if (p.q_stride_tok % epl || p.q_stride_tok < (int64_t)p.Hq * D ||
      (((uintptr_t)p.q | (uintptr_t)p.q_out | (uintptr_t)p.cos | (uintptr_t)p.sin) & 15))
    return fail(MI355_EINVAL, "%s: rows must be 16-byte aligned and a token's heads packed", what);
  if (p.slots && (p.k_stride_tok % epl || p.v_stride_tok % epl || p.k_stride_tok < (int64_t)p.Hkv * D ||
                  p.v_stride_tok < (int64_t)p.Hkv * D || (((uintptr_t)p.k | (uintptr_t)p.v) & 15)))
    return fail(MI355_EINVAL, "%s: key / value rows must be 16-byte aligned and a token's heads packed", what);
  const int64_t eb = dtype == MI355_F32 ? 4 : 2, out_bytes = (int64_t)T * p.Hq * D * eb;
  if (T > 0 && (kv4_overlaps(p.q_out, out_bytes, p.q, p.q_stride_tok * eb, p.Hq * D * eb, T) ||
                (p.slots && (kv4_overlaps(p.q_out, out_bytes, p.k, p.k_stride_tok * eb, p.Hkv * D * eb, T) ||
                             kv4_overlaps(p.q_out, out_bytes, p.v, p.v_stride_tok * eb, p.Hkv * D * eb, T)))))
    return fail(MI355_EINVAL, "%s: the output overlaps the rows it is made from", what);
  if (rotary_dim == 0) p.cos = p.sin = nullptr;
  p.R = rotary_dim;
  p.heads = p.slots ? p.Hq + 2 * p.Hkv : p.Hq;
  p.T = T;
  if (!kv4_grid_ok(ceil_div64((int64_t)T * p.heads, 256 / (D / 8)), 256)) return fail(MI355_EINVAL, "%s: too many rows (T=%d)", what, T);
  switch (dtype) {
    case MI355_F32: return launch_append<F32>(p, D, interleaved != 0, s);
    case MI355_BF16: return launch_append<BF16>(p, D, interleaved != 0, s);
    default: return launch_append<F16>(p, D, interleaved != 0, s);
  }
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_rope_angles(float* cos_out, float* sin_out, const int64_t* positions, const double* inv_freq,
                                 double factor, int32_t T, int32_t half_dim, void* stream) {
  if (T == 0) return 0;
  if (!cos_out || !sin_out || !positions || !inv_freq) return fail(MI355_EINVAL, "rope_angles: null pointer");
  if (T < 0 || half_dim <= 0) return fail(MI355_EINVAL, "rope_angles: bad shape (T=%d half_dim=%d)", T, half_dim);
  const int64_t total = (int64_t)T * half_dim;
  if (!kv4_grid_ok(ceil_div64(total, 256), 256)) return fail(MI355_EINVAL, "rope_angles: too many rows (T=%d)", T);
  hipLaunchKernelGGL(rope_angles_kernel, dim3((unsigned)ceil_div64(total, 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), cos_out, sin_out, positions, inv_freq, factor, total, half_dim);
  return check_launch("rope_angles_kernel");
}

extern "C" int mi355_rope_rotate(void* out, const void* x, int64_t x_stride_tok, const float* cos_rows,
                                 const float* sin_rows, int32_t rotary_dim, int32_t interleaved, int32_t T, int32_t H,
                                 int32_t D, int32_t dtype, void* stream) {
  if (T == 0) return 0;
  if (!out || !x) return fail(MI355_EINVAL, "rope_rotate: null pointer");
  AppendParams4 p{};
  p.q = static_cast<const char*>(x);
  p.q_out = static_cast<char*>(out);
  p.q_stride_tok = x_stride_tok;
  p.cos = cos_rows;
  p.sin = sin_rows;
  p.Hq = H;
  return append_impl("rope_rotate", p, T, D, rotary_dim, interleaved, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int mi355_rope_kv4_write(void* q_out, const void* q, const void* k, const void* v, int64_t q_stride_tok,
                                    int64_t k_stride_tok, int64_t v_stride_tok, const float* cos_rows,
                                    const float* sin_rows, int32_t rotary_dim, int32_t interleaved,
                                    const int64_t* slots, void* k_cache, void* v_cache, int32_t T, int32_t Hq,
                                    int32_t Hkv, int32_t D, int32_t block_size, int32_t num_blocks,
                                    int64_t stride_block, int64_t stride_head, int32_t dtype, void* stream) {
  if (T == 0) return 0;
  if (!q_out || !q || !k || !v || !slots) return fail(MI355_EINVAL, "rope_kv4_write: null pointer");
  if (int rc = kv4_check_cache("rope_kv4_write", k_cache, v_cache, Hkv, D, block_size, num_blocks, stride_block, stride_head))
    return rc;
  AppendParams4 p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.q_out = static_cast<char*>(q_out);
  p.q_stride_tok = q_stride_tok;
  p.k_stride_tok = k_stride_tok;
  p.v_stride_tok = v_stride_tok;
  p.cos = cos_rows;
  p.sin = sin_rows;
  p.slots = slots;
  p.cache = kv4_cache(k_cache, v_cache, stride_block, stride_head, num_blocks, block_size / kKv4Tile);
  p.num_slots = (int64_t)num_blocks * block_size;
  p.bs_shift = ilog2_exact(block_size);
  p.Hq = Hq;
  p.Hkv = Hkv;
  return append_impl("rope_kv4_write", p, T, D, rotary_dim, interleaved, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int mi355_kv4_read_slots(void* k_out, void* v_out, const void* k_cache, const void* v_cache,
                                    const int64_t* slots, int32_t T, int32_t Hkv, int32_t D, int32_t block_size,
                                    int32_t num_blocks, int64_t stride_block, int64_t stride_head, int32_t dtype,
                                    void* stream) {
  if (T == 0) return 0;
  if (!k_out || !v_out || !slots) return fail(MI355_EINVAL, "kv4_read_slots: null pointer");
  if (int rc = kv4_check_cache("kv4_read_slots", k_cache, v_cache, Hkv, D, block_size, num_blocks, stride_block, stride_head))
    return rc;
  if (T < 0) return fail(MI355_EINVAL, "kv4_read_slots: bad shape (T=%d)", T);
  if (!kv4_dtype_ok(dtype)) return fail(MI355_EINVAL, "kv4_read_slots: dtype %d", dtype);
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return fail(MI355_EINVAL, "kv4_read_slots: outputs must be 16-byte aligned");
  ReadParams4 p{};
  p.k_out = static_cast<char*>(k_out);
  p.v_out = static_cast<char*>(v_out);
  p.slots = slots;
  p.cache = kv4_cache(k_cache, v_cache, stride_block, stride_head, num_blocks, block_size / kKv4Tile);
  p.T = T;
  p.num_slots = (int64_t)num_blocks * block_size;
  p.Hkv = Hkv;
  p.bs_shift = ilog2_exact(block_size);
  if (!kv4_grid_ok(ceil_div64((int64_t)T * 2 * Hkv, 256 / (D / 8)), 256)) return fail(MI355_EINVAL, "kv4_read_slots: too many rows (T=%d)", T);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MI355_F32: return launch_read<F32>(p, D, s);
    case MI355_BF16: return launch_read<BF16>(p, D, s);
    default: return launch_read<F16>(p, D, s);
  }
}
