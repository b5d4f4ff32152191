// Attention of several new query tokens per sequence over the 4-bit KV cache (their K / V rows are in
// it already): query j of a segment attends to positions 0 .. pos0 + j.
//
// The query rows of a (segment, kv head) are its (token, query head of the group) pairs; they are the
// columns of a score tile S^T = K Q^T, whose weights go back into the matrix unit in the registers they
// were born in (see kv4.h).  Conversion of codes to bf16 (exact up to the largest bf16) is what the format costs beside attention
// in bf16 -- 130 vector instructions per 32 tokens of 128 dims, as many as the softmax of 32 columns -- and
// the two kernels differ in who does it:
//   kv4_prefill_kernel  many rows.  A workgroup of four waves owns four tiles of 16 or 32 columns and walks
//       the context in stages of SUB steps of 32 tokens.  Per stage each wave converts a quarter of the K
//       and V codes and leaves them in LDS as the operands of the matrix instruction; every wave reads them
//       all back.  Codes travel from memory one stage ahead in registers, operands one stage ahead in LDS
//       (two buffers, one barrier per stage).  The matrix pipe is busy for 48 % of its time at 128 dims, and
//       vector instructions (conversion, softmax, the weights' second piece) take turns with it.
//   kv4_rows_kernel     few rows.  A workgroup owns 32 or 64 columns, its four or eight waves take the steps in turn
//       and convert their own in registers: no barrier, short walks, more conversion per row.
#include <algorithm>
#include <cmath>

#include "kv4.h"

namespace mi355 {
namespace {

constexpr int kWaves = 4;

// How a stage is cut: steps per stage, and the part of it each of the four waves converts -- NB V blocks
// of one step, and K operands [first, first + KF) of KT tiles.
template <int D>
struct Stage {
  static constexpr int KS = D / 32;
  static constexpr int SUB = D == 256 ? 1 : D == 32 ? 4 : 2;
  static constexpr int NB = D <= 64 ? 1 : 2;
  static constexpr int KT = D == 32 ? 2 : 1, KF = D <= 64 ? KS : 4;
  static constexpr int kTokens = SUB * kKv4Step;
  static __device__ __forceinline__ int step(int w) { return D == 256 ? 0 : D == 32 ? w : w / 2; }
  static __device__ __forceinline__ int v_block(int w) { return D == 256 ? 2 * w : D == 32 ? 0 : NB * (w & 1); }
  static __device__ __forceinline__ int k_tile(int w) { return D == 256 ? w / 2 : D == 32 ? 0 : w & 1; }   // (the first of KT)
  static __device__ __forceinline__ int k_first(int w) { return D == 256 ? 4 * (w & 1) : 0; }
};

struct Kv4PrefillParams {
  char* out;
  const char* q;
  Kv4Cache cache;
  const int32_t* bt;
  const int32_t* seg_q0;
  const int32_t* seg_len;
  const int32_t* seg_pos0;
  int64_t q_stride;   // elements
  float* ws;   // [total rows * Hq][nsplit][D + 4]: unnormalised sums, running maximum, sum of weights
  int nseg, total_rows, max_q_len, Hq, Hkv, G, max_blocks, max_ctx, row_tiles, nsplit, tps /* tokens per split, whole stages */;
  float scale2, raise;   // |scale| * log2(e); kKv4Raise in units of a raw score
  int flip;              // a negative scale: the queries are negated
};

// Rows of a segment; none outside the tensors, whatever the segment says.
__device__ __forceinline__ int segment_rows(const Kv4PrefillParams& p, int q0, int len) {
  return q0 < 0 || q0 >= p.total_rows ? 0 : min(min(len, p.max_q_len), p.total_rows - q0);
}

// Between two waves' uses of LDS; global loads may stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// How a wave lays out its tile of COLS query rows (a lane's column is lane % COLS): with 16 columns the 16x16x32 matrix
// instruction, scores and values of 16 rows at a time; with 32 the 32x32x16 one.
//   scores   32 tokens of a step in rows; a lane holds TOK of them.  With 32 columns row R is token (R & 7) + 8 (R >> 4) of
//            tile (R >> 3) & 1, which makes the lane's tokens the ones that one conversion of a value block yields.
//   values   32 dims of a block in rows: two tiles of even and odd dims, or one tile with the odd dims behind the even ones
template <int COLS>
struct Layout;
template <>
struct Layout<16> {
  static constexpr int kTok = 8, kQ = 1, kHalf = 1;   // tokens per lane; contraction steps of a value product; chunks of 8 dims per block
  typedef f32x4 scores_t[2];
  typedef f32x4 sums_t[2];
  static __device__ __forceinline__ int token(int g, int e) { return (e >> 2) * kKv4Tile + 4 * g + (e & 3); }
  // where the frag of tile t, token c, dims (g, s) goes (units of operands of 64 lanes, and the lane)
  static __device__ __forceinline__ int k_slot(int lane, int t, int KS) { return t * KS * 64 + lane; }
  static constexpr int kStepS = 64;   // from s to s + 1
  static __device__ __forceinline__ int v_even(int lane) { return lane; }
  static __device__ __forceinline__ int v_odd(int lane) { return 64 + lane; }
  static __device__ __forceinline__ int q_dim(int D, int g, int f) { return g * (D / 4) + 8 * f; }
  static __device__ __forceinline__ float score(const scores_t& S, int e) { return S[e >> 2][e & 3]; }
  static __device__ __forceinline__ int chunk(int g, int) { return 8 * g; }
  static __device__ __forceinline__ float even(const sums_t& a, int, int i) { return a[0][i]; }
  static __device__ __forceinline__ float odd(const sums_t& a, int, int i) { return a[1][i]; }
};
template <>
struct Layout<32> {
  static constexpr int kTok = 16, kQ = 2, kHalf = 2;
  typedef f32x16 scores_t[1];
  typedef f32x16 sums_t[1];
  static __device__ __forceinline__ int token(int g, int e) { return ((e >> 2) & 1) * kKv4Tile + (e >> 3) * 8 + 4 * g + (e & 3); }
  static __device__ __forceinline__ int k_slot(int lane, int t, int) {
    const int g = lane >> 4, c = lane & 15;
    return (g >> 1) * 64 + (g & 1) * 32 + (c >> 3) * 16 + t * 8 + (c & 7);
  }
  static constexpr int kStepS = 128;
  static __device__ __forceinline__ int v_even(int lane) { return (lane >> 5) * 64 + ((lane >> 4) & 1) * 32 + (lane & 15); }
  static __device__ __forceinline__ int v_odd(int lane) { return v_even(lane) + 16; }
  static __device__ __forceinline__ int q_dim(int D, int g, int f) { return (2 * (f & 1) + g) * (D / 4) + 8 * (f >> 1); }
  static __device__ __forceinline__ float score(const scores_t& S, int e) { return S[0][e]; }
  static __device__ __forceinline__ int chunk(int g, int h) { return 16 * h + 8 * g; }
  static __device__ __forceinline__ float even(const sums_t& a, int h, int i) { return a[0][4 * h + i]; }
  static __device__ __forceinline__ float odd(const sums_t& a, int h, int i) { return a[0][8 + 4 * h + i]; }
};
__device__ __forceinline__ f32x16 mfma32_bf16(bf16x8_t a, bf16x8_t b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <class Tag, int D, int COLS>
__global__ void __launch_bounds__(256, 2) kv4_prefill_kernel(const Kv4PrefillParams p) {
  typedef Stage<D> St;
  typedef Layout<COLS> Lay;
  constexpr int NP = Kv4Pieces<Tag>::n, NW = Kv4Pieces<Tag>::weights, KS = D / 32, EB = Tag::kBytes;
  constexpr int SUB = St::SUB, NB = St::NB, KT = St::KT, KF = St::KF;
  constexpr int KA = KS < 4 ? KS : 4, VA = KS < 2 ? KS : 2;   // operands read ahead of their use
  constexpr int TOK = Lay::kTok, NQ = Lay::kQ, QF = KS * NQ;
  __shared__ bf16x8_t s_k[2][SUB][2 * KS * 64], s_v[2][SUB][KS][2 * 64];
  __shared__ uint32_t s_nan[2][SUB][KS];   // tokens of a step whose V block was NaN (masked stages only)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane / COLS, col = lane % COLS;
  int idx = blockIdx.x;
  const int h = idx % p.Hkv;   // (kv heads on neighbouring XCDs: the row tiles of one head share an L2 where Hkv is a multiple of 8)
  idx /= p.Hkv;
  const int seg = idx % p.nseg;
  const int rt = p.row_tiles - 1 - idx / p.nseg;   // the longest contexts first
  const int q0 = p.seg_q0[seg], pos0 = p.seg_pos0[seg], len = segment_rows(p, q0, p.seg_len[seg]);
  const int rows = len * p.G, wg_row0 = rt * kWaves * COLS;
  if (wg_row0 >= rows) return;
  const int row0 = wg_row0 + wave * COLS;

  int lim;        // last position the column attends to; -1: none
  int64_t orow;   // its row of out (and of q), -1: none
  bf16x8_t qf[QF][NP];
  {
    const int r = row0 + col, rr = min(r, rows - 1);
    const int tok = rr / p.G, hq = h * p.G + rr % p.G;
    lim = min(pos0 + tok, p.max_ctx - 1);
    orow = r < rows ? (int64_t)(q0 + tok) * p.Hq + hq : -1;
    const char* src = p.q + ((int64_t)(q0 + tok) * p.q_stride + (int64_t)hq * D) * EB;
#pragma unroll
    for (int f = 0; f < QF; ++f) {
      float x[8];
      load8<Tag>(src + Lay::q_dim(D, g, f) * EB, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = p.flip ? -x[e] : x[e];
      bf16_pieces<NP>(x, qf[f]);
    }
  }
  auto limit = [&](int r) { return min(pos0 + min(r, rows - 1) / p.G, p.max_ctx - 1); };
  const int wave_first = limit(row0);
  const int wg_first = limit(wg_row0), wg_last = limit(wg_row0 + kWaves * COLS - 1);
  const int wave_last = row0 < rows ? limit(row0 + COLS - 1) : -1;

  typename Lay::sums_t acc[KS];
  float m = kKv4Floor;   // running maximum of the raw scores
  float sum = 0.f;       // of the lane's weights
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (auto& a : acc[s]) a = 0.f;

  // ---- this wave's part of a stage
  const int32_t* table = p.bt + (int64_t)seg * p.max_blocks;
  const int last_tile = max(wg_last, 0) / kKv4Tile;
  const int vstep = St::step(wave), vblk = St::v_block(wave), kstep = vstep, ktile = St::k_tile(wave),
            kfirst = St::k_first(wave);
  const int k_slot = Lay::k_slot(lane, St::k_tile(wave), KS), v_even = Lay::v_even(lane), v_odd = Lay::v_odd(lane);
  uint32_t o_k, o_ks, o_v, o_vs, turn;   // the lane's places in a record
  {
    Kv4Lane<D> at(lane);
    o_k = at.k + 4 * kfirst;
    o_ks = at.ks;
    o_v = at.v + 4 * vblk;
    o_vs = at.vs + 4 * vblk;
    turn = D == 256 && kfirst ? (at.turn + 8) & 31 : at.turn;
  }
  uint32_t rk[KT][KF], rks[KT], rv[2][NB], rvs[2][NB];
  const char* const kbase = p.cache.k + (int64_t)h * p.cache.s_head;
  const char* const vbase = p.cache.v + (int64_t)h * p.cache.s_head;
  static_assert(KT == 2 || KT == 1, "");
  Kv4Place n0{}, n1{};   // the next stage's records (of the step this wave converts), asked for a stage ahead
  auto place = [&](int t0) {
    const int tile = (int)((uint32_t)(t0 + vstep * kKv4Step) / kKv4Tile);
    n0 = kv4_place(p.cache, table, min(tile, last_tile));
    n1 = kv4_place(p.cache, table, min(tile + 1, last_tile));
  };
  auto fetch = [&]() {
    const int64_t r0 = kv4_record(p.cache, n0, kv4_tile_bytes(D)), r1 = kv4_record(p.cache, n1, kv4_tile_bytes(D));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      gptr rec = scalar_base(vbase + (i ? r1 : r0));
      load_words<false>(rec + lane_offset(o_v), rv[i]);
      load_words<false>(rec + lane_offset(o_vs), rvs[i]);
    }
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      gptr rec = scalar_base(kbase + ((KT == 2 ? i : ktile) ? r1 : r0));
      uint32_t w[1];
      load_words<false>(rec + lane_offset(o_k), rk[i]);
      load_words<false>(rec + lane_offset(o_ks), w);
      rks[i] = w[0];
    }
  };
  // Codes in registers -> operands in LDS, for the stage that starts at token t0.
  auto convert = [&](int t0, int buf) {
    if (t0 + St::kTokens - 1 > wg_first) {
      // Some column must not see some of these value rows; they enter its product with weight 0, and 0 * NaN is
      // NaN.  Rows behind the workgroup's last position count as 0; NaN blocks become 0 here and are put back,
      // for the columns that see them, where the stage is used.  (Scale bytes above the largest that the append
      // writes count as NaN here: with them a value may be an infinity.)
      uint32_t nan[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) nan[b] = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // (of this lane's four tokens: those of the record's order, whatever the number of columns)
        const int live = wg_last + 1 - (t0 + vstep * kKv4Step + i * kKv4Tile + 4 * (lane >> 4));
        const uint32_t keep = live >= 4 ? ~0u : (live <= 0 ? 0u : (1u << (8 * live)) - 1u);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t vs = (rvs[i][b] & keep) | (0x7f7f7f7fu & ~keep), bad = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool is_nan = ((vs >> (8 * j)) & 0xffu) > kKv4MaxExp + 127u;
            const uint64_t all = __ballot(is_nan);   // lanes 0, 16, 32, 48 speak for tokens j, 4 + j, 8 + j, 12 + j
            nan[b] |= (uint32_t)((all & 1) | (all >> 16 & 1) << 4 | (all >> 32 & 1) << 8 | (all >> 48 & 1) << 12) << (16 * i + j);
            bad |= is_nan ? 0xffu << (8 * j) : 0u;
          }
          rv[i][b] &= keep & ~bad;
          rvs[i][b] = (vs & ~bad) | (0x7f7f7f7fu & bad);
        }
      }
      if (lane == 0) {
#pragma unroll
        for (int b = 0; b < NB; ++b) s_nan[buf][vstep][vblk + b] = nan[b];
      }
    }
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const float sc = u2f(__builtin_amdgcn_alignbit(rks[i], rks[i], turn));
      const int slot = KT == 2 ? Lay::k_slot(lane, i, KS) : k_slot;
#pragma unroll
      for (int f = 0; f < KF; ++f) s_k[buf][kstep][slot + (kfirst + f) * Lay::kStepS] = kv4_k_frag(rk[i][f], sc);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      bf16x8_t ev, od;
      kv4_v_frags(rv[0][b], rv[1][b], rvs[0][b], rvs[1][b], ev, od);
      s_v[buf][vstep][vblk + b][v_even] = ev;
      s_v[buf][vstep][vblk + b][v_odd] = od;
    }
  };

  if (wg_last >= 0) {
    place(0);
    fetch();
    place(St::kTokens);
    convert(0, 0);
    fetch();
    place(2 * St::kTokens);
    int buf = 0;
    for (int t0 = 0; t0 <= wg_last; t0 += St::kTokens, buf ^= 1) {
      lds_barrier();
      convert(t0 + St::kTokens, buf ^ 1);   // (behind the last stage: the last tile again, read by nobody)
      fetch();
      place(min(t0 + 3 * St::kTokens, wg_last));
      const bool wg_masked = t0 + St::kTokens - 1 > wg_first;
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        const int ts = t0 + sub * kKv4Step;
        if (ts > wave_last) break;
        const bool masked = ts + kKv4Step - 1 > wave_first;
        typename Lay::scores_t S;
#pragma unroll
        for (auto& c : S) c = 0.f;
        bf16x8_t kf[2][KA];   // K operands, read 2 KA ahead
#pragma unroll
        for (int f = 0; f < 2 * KA; ++f) kf[f / KA][f % KA] = s_k[buf][sub][f * 64 + lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < 2 * KS; ++f) {
          const bf16x8_t a = kf[f / KA % 2][f % KA];
          if (f + 2 * KA < 2 * KS) kf[f / KA % 2][f % KA] = s_k[buf][sub][(f + 2 * KA) * 64 + lane];
#pragma unroll
          for (int n = 0; n < NP; ++n) {
            if constexpr (COLS == 16) S[f / KS] = mfma_bf16(a, qf[f % KS][n], S[f / KS]);
            else S[0] = mfma32_bf16(a, qf[f][n], S[0]);
          }
        }
        bf16x8_t vf[VA][2];   // V operands of the first blocks, on their way during the softmax
#pragma unroll
        for (int s = 0; s < VA; ++s) {
          vf[s][0] = s_v[buf][sub][s][lane];
          vf[s][1] = s_v[buf][sub][s][64 + lane];
        }
        __builtin_amdgcn_sched_barrier(0);
        if (wg_masked) {
          const int seen = lim + 1 - ts;   // tokens of the step the column sees
          const uint32_t sees = seen >= 32 ? ~0u : (seen <= 0 ? 0u : (1u << seen) - 1u);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const uint32_t nan = __builtin_amdgcn_readfirstlane(s_nan[buf][sub][s]);
            if (nan & sees) {
#pragma unroll
              for (auto& a : acc[s]) a = __builtin_nanf("");
            }
          }
        }
        float x[TOK];
#pragma unroll
        for (int e = 0; e < TOK; ++e) x[e] = Lay::score(S, e);
        if (masked) {
#pragma unroll
          for (int e = 0; e < TOK; ++e)
            if (ts + Lay::token(g, e) > lim) x[e] = -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e + 1 < TOK; e += 2) top = fmaxf(fmaxf(top, x[e]), x[e + 1]);
        top = fmaxf(top, x[TOK - 1]);
        if (__ballot(top > m + p.raise)) {
          if constexpr (COLS == 16) top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float mn = fmaxf(m, top), f = kv4_shift(m, mn, p.scale2);
          m = mn;
          sum *= f;
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (auto& a : acc[s]) a *= f;
        }
        bf16x8_t pf[NQ][NW];
#pragma unroll
        for (int e = 0; e < TOK; ++e) {
          x[e] = kv4_weight(x[e], m, p.scale2);
          sum += x[e];
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) weight_pieces<NW>(*reinterpret_cast<const float(*)[8]>(&x[8 * n]), pf[n]);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const bf16x8_t a0 = vf[s % VA][0], a1 = vf[s % VA][1];
          if (s + VA < KS) {
            vf[s % VA][0] = s_v[buf][sub][s + VA][lane];
            vf[s % VA][1] = s_v[buf][sub][s + VA][64 + lane];
          }
#pragma unroll
          for (int n = 0; n < NW; ++n) {
            if constexpr (COLS == 16) {
              acc[s][0] = mfma_bf16(a0, pf[0][n], acc[s][0]);
              acc[s][1] = mfma_bf16(a1, pf[0][n], acc[s][1]);
            } else {
              acc[s][0] = mfma32_bf16(a0, pf[0][n], acc[s][0]);
              acc[s][0] = mfma32_bf16(a1, pf[1][n], acc[s][0]);
            }
          }
        }
      }
    }
  }

  if constexpr (COLS == 16) sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (orow < 0) return;
  const float inv = lim >= 0 ? 1.f / sum : 0.f;   // a query before position 0 sees nothing: zeros
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int c = 0; c < Lay::kHalf; ++c) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = lim >= 0 ? Lay::even(acc[s], c, i) * inv : 0.f;
        x[2 * i + 1] = lim >= 0 ? Lay::odd(acc[s], c, i) * inv : 0.f;
      }
      store8<Tag>(p.out + (orow * D + 32 * s + Lay::chunk(g, c)) * EB, x);
    }
}

// A workgroup of CT tiles of 32 query rows; its W waves take the steps of the context in turn, so that a walk is 1 / W
// as long.  A wave converts its own steps in registers, as decode does, in the lanes where the matrix instruction wants them:
//   K  lane (g, R) holds token (R & 7) + 8 (R >> 4) of tile (R >> 3) & 1, dims of groups g and 2 + g
//   V  lane (g, half, c) holds dims 2 c, 2 c + 1 of a block of its half of the blocks, tokens of groups g and 2 + g; the even
//      dims of two blocks are the 32 rows of one product, the odd dims of another (head_dim 32: both of the only block)
// The queries wait in LDS, where the waves' sums meet at the end.
template <class Tag, int D, int CT, int W>
__global__ void __launch_bounds__(W * 64, 2) kv4_rows_kernel(const Kv4PrefillParams p) {
  constexpr int NP = Kv4Pieces<Tag>::n, NW = Kv4Pieces<Tag>::weights, KS = D / 32, EB = Tag::kBytes, QF = 2 * KS;
  constexpr int QD = QF < 4 ? QF : NP == 1 && D < 256 && CT == 1 ? 4 : 2;   // query operands read ahead
  constexpr int VB = KS > 1 ? KS / 2 : 1;            // value blocks per lane
  constexpr int NT = KS > 1 ? 2 * VB : 1;            // 32-row tiles of the output
  constexpr int kPart = D < 128 ? D : 128, kParts = D / kPart;   // dims of an epilogue pass
  constexpr int kRow = kPart + 4, ROWS = CT * 32;
  constexpr int kQ = CT * QF * NP * 64 * 16, kJoin = W * 32 * kRow * 4;
  __shared__ __attribute__((aligned(16))) char s_mem[kQ > kJoin ? kQ : kJoin];
  bf16x8_t* const s_q = reinterpret_cast<bf16x8_t*>(s_mem);   // [CT][QF][NP][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5, col = lane & 31, half = col >> 4, c = lane & 15;
  int idx = blockIdx.x;
  const int h = idx % p.Hkv;   // (as above; and a split that is empty in some segments would leave whole XCDs idle)
  idx /= p.Hkv;
  const int sp = idx % p.nsplit;
  idx /= p.nsplit;
  const int seg = idx % p.nseg;
  const int rt = p.row_tiles - 1 - idx / p.nseg;
  const int q0 = p.seg_q0[seg], pos0 = p.seg_pos0[seg], len = segment_rows(p, q0, p.seg_len[seg]);
  const int rows = len * p.G, row0 = rt * ROWS;
  if (row0 >= rows) return;
  auto limit = [&](int r) { return min(pos0 + min(r, rows - 1) / p.G, p.max_ctx - 1); };
  const int wg_first = limit(row0), wg_end = limit(row0 + ROWS - 1);
  const int lo = sp * p.tps, wg_last = min(wg_end, lo + p.tps - 1);
  if (lo > wg_last && sp > 0) return;

  // queries -> LDS, as the operands the waves read
  int lim[CT];   // last position the column attends to; negative: none
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    lim[ct] = limit(row0 + ct * 32 + col);
    const int r = min(row0 + ct * 32 + col, rows - 1), tok = r / p.G, hq = h * p.G + r % p.G;
    const char* src = p.q + ((int64_t)(q0 + tok) * p.q_stride + (int64_t)hq * D) * EB;
    for (int f = wave; f < QF; f += W) {
      float x[8];
      load8<Tag>(src + ((2 * (f & 1) + g) * (D / 4) + 8 * (f >> 1)) * EB, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = p.flip ? -x[e] : x[e];
      bf16x8_t y[NP];
      bf16_pieces<NP>(x, y);
#pragma unroll
      for (int n = 0; n < NP; ++n) s_q[((ct * QF + f) * NP + n) * 64 + lane] = y[n];
    }
  }

  f32x16 acc[CT][NT];
  float m[CT], sum[CT];   // running maximum of the raw scores; sum of the lane's weights
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = kKv4Floor;
    sum[ct] = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[ct][j] = 0.f;
  }

  const int32_t* table = p.bt + (int64_t)seg * p.max_blocks;
  const int last_tile = max(wg_last, 0) / kKv4Tile;
  const char* const kbase = p.cache.k + (int64_t)h * p.cache.s_head;
  const char* const vbase = p.cache.v + (int64_t)h * p.cache.s_head;
  Kv4Place n0{}, n1{};
  auto place = [&](int t0) {
    const int tile = (int)((uint32_t)t0 / kKv4Tile);
    n0 = kv4_place(p.cache, table, min(tile, last_tile));
    n1 = kv4_place(p.cache, table, min(tile + 1, last_tile));
  };
  // K: lane (g, R) holds token (R & 7) + 8 (R >> 4) of tile (R >> 3) & 1, dims of groups g and 2 + g
  constexpr int KW = D / 32, SW = D == 256 ? 2 : 1;
  const int ktok = (col & 7) + 8 * half;
  const bool ktile = (col >> 3) & 1;
  const uint32_t o_k = ktok * (D / 2) + g * (D / 8);
  const int sbyte = ktok * (D / 32) + (D == 256 ? 2 * g : D == 128 ? g : 0);   // of group g, s = 0
  const uint32_t o_ks = 8 * D + (D == 256 ? ktok * 8 : (sbyte & ~3)), turn = 9 + 8 * (sbyte & 3);
  uint32_t o_v = ((g * 16 + c) * KS + (KS > 1 ? half * VB : 0)) * 4, o_vs = 8 * D + (g * KS + (KS > 1 ? half * VB : 0)) * 4;
  uint32_t rk[2][KW], rks[SW], rv[2][2][VB], rvs[2][2][VB];
  auto fetch_k = [&](int64_t r0, int64_t r1) {
    const gptr rec = (gptr)kbase + (ktile ? r1 : r0);
    load_words<false>(rec + o_k, rk[0]);
    load_words<false>(rec + o_k + D / 4, rk[1]);
    load_words<false>(rec + o_ks, rks);
  };
  auto fetch_v = [&](int64_t r0, int64_t r1) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      gptr rec = scalar_base(vbase + (t ? r1 : r0));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        load_words<false>(rec + lane_offset(o_v) + q * 64 * D / 16, rv[t][q]);
        load_words<false>(rec + lane_offset(o_vs) + q * 2 * KS * 4, rvs[t][q]);
      }
    }
  };
  auto k_scale = [&](int f) {
    const int pt = f & 1, s = f >> 1;
    if constexpr (D == 256) return u2f(__builtin_amdgcn_alignbit(rks[pt], rks[pt], turn + 8 * (s >> 2)));
    return u2f(__builtin_amdgcn_alignbit(rks[0], rks[0], turn + pt * (D == 128 ? 16 : D == 64 ? 8 : 0)));
  };
  __syncthreads();

  constexpr int kStride = W * kKv4Step;
  int t0 = lo + wave * kKv4Step;
  if (t0 <= wg_last) {
    place(t0);
    const int64_t r0 = kv4_record(p.cache, n0, kv4_tile_bytes(D)), r1 = kv4_record(p.cache, n1, kv4_tile_bytes(D));
    fetch_k(r0, r1);
    fetch_v(r0, r1);
    place(min(t0 + kStride, wg_last));
  }
  // One step; its registers are refilled for the next as soon as their codes are converted.
  auto step = [&]() {
    const int64_t r0 = kv4_record(p.cache, n0, kv4_tile_bytes(D)), r1 = kv4_record(p.cache, n1, kv4_tile_bytes(D));
    const bool masked = t0 + kKv4Step - 1 > wg_first;
    if (masked) {
      uint32_t nan[VB];
#pragma unroll
      for (int b = 0; b < VB; ++b) nan[b] = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int live = wg_last + 1 - (t0 + t * kKv4Tile + 4 * (g + 2 * q));
          const uint32_t keep = live >= 4 ? ~0u : (live <= 0 ? 0u : (1u << (8 * live)) - 1u);
#pragma unroll
          for (int b = 0; b < VB; ++b) {
            const uint32_t vs = (rvs[t][q][b] & keep) | (0x7f7f7f7fu & ~keep);
            uint32_t bad = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bool is_nan = ((vs >> (8 * j)) & 0xffu) > kKv4MaxExp + 127u;
              bad |= is_nan ? 0xffu << (8 * j) : 0u;
              nan[b] |= is_nan ? 1u << (t * 16 + 4 * (g + 2 * q) + j) : 0u;
            }
            rv[t][q][b] &= keep & ~bad;
            rvs[t][q][b] = (vs & ~bad) | (0x7f7f7f7fu & bad);
          }
        }
#pragma unroll
      for (int b = 0; b < VB; ++b) {
        nan[b] |= __shfl_xor(nan[b], 32);   // all tokens; by halves of the lanes the two blocks
        const uint32_t mine = nan[b], other = __shfl_xor(mine, 16);
        if (__ballot(mine | other)) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            const int seen = lim[ct] + 1 - t0;   // tokens of the step the column sees
            const uint32_t sees = seen >= 32 ? ~0u : (seen <= 0 ? 0u : (1u << seen) - 1u);
            const bool low = ((half ? other : mine) & sees) != 0, high = ((half ? mine : other) & sees) != 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {   // (rows 16 .. 31, the second half's blocks, are elements 8 .. 15)
              const bool hit = KS > 1 && e >= 8 ? high : low;
              acc[ct][NT > 1 ? 2 * b : 0][e] = hit ? __builtin_nanf("") : acc[ct][NT > 1 ? 2 * b : 0][e];
              if constexpr (NT > 1) acc[ct][2 * b + 1][e] = hit ? __builtin_nanf("") : acc[ct][2 * b + 1][e];
            }
          }
        }
      }
    }
    f32x16 S[CT];
    bf16x8_t qr[QD][CT][NP];
    auto read_q = [&](int f) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int n = 0; n < NP; ++n) qr[f % QD][ct][n] = s_q[((ct * QF + f) * NP + n) * 64 + lane];
    };
#pragma unroll
    for (int f = 0; f < QD; ++f) read_q(f);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) S[ct] = 0.f;
#pragma unroll
    for (int f = 0; f < QF; ++f) {
      const bf16x8_t a = kv4_k_frag(rk[f & 1][f >> 1], k_scale(f));
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int n = 0; n < NP; ++n) S[ct] = mfma32_bf16(a, qr[f % QD][ct][n], S[ct]);
      if (f + QD < QF) read_q(f + QD);
      __builtin_amdgcn_sched_barrier(0);
    }
    fetch_k(r0, r1);
    place(min(t0 + 2 * kStride, wg_last));
    bf16x8_t pf[CT][2][NW];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if (masked) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (t0 + Layout<32>::token(g, e) > lim[ct]) S[ct][e] = -INFINITY;
      }
      float top = S[ct][0];
#pragma unroll
      for (int e = 1; e + 1 < 16; e += 2) top = fmaxf(fmaxf(top, S[ct][e]), S[ct][e + 1]);
      top = fmaxf(top, S[ct][15]);
      if (__ballot(top > m[ct] + p.raise)) {
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m[ct], top), f = kv4_shift(m[ct], mn, p.scale2);
        m[ct] = mn;
        sum[ct] *= f;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[ct][j] *= f;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = kv4_weight(S[ct][8 * n + e], m[ct], p.scale2);
          sum[ct] += x[e];
        }
        weight_pieces<NW>(x, pf[ct][n]);
      }
    }
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        bf16x8_t ev, od;
        kv4_v_frags(rv[0][q][b], rv[1][q][b], rvs[0][q][b], rvs[1][q][b], ev, od);
        if constexpr (KS == 1) ev = half ? od : ev;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int n = 0; n < NW; ++n) {
            acc[ct][NT > 1 ? 2 * b : 0] = mfma32_bf16(ev, pf[ct][q][n], acc[ct][NT > 1 ? 2 * b : 0]);
            if constexpr (NT > 1) acc[ct][2 * b + 1] = mfma32_bf16(od, pf[ct][q][n], acc[ct][2 * b + 1]);
          }
      }
    fetch_v(r0, r1);
    t0 += kStride;
  };
  while (t0 <= wg_last) step();

  // join the waves
  float* const s_o = reinterpret_cast<float*>(s_mem) + wave * 32 * kRow;
  constexpr int P = kPart / 8;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float total = sum[ct] + __shfl_xor(sum[ct], 32);
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      __syncthreads();
      float* const row = s_o + col * kRow;
#pragma unroll
      for (int j = 0; j < VB; ++j)
#pragma unroll
        for (int hf = 0; hf < (KS > 1 ? 2 : 1); ++hf) {
          const int blk = j + hf * VB;
          if (blk * 32 / kPart != part) continue;
#pragma unroll
          for (int bl = 0; bl < 2; ++bl) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (KS > 1) {
                x[2 * i] = acc[ct][2 * j][(2 * hf + bl) * 4 + i];
                x[2 * i + 1] = acc[ct][2 * j + 1][(2 * hf + bl) * 4 + i];
              } else {
                x[2 * i] = acc[ct][0][bl * 4 + i];
                x[2 * i + 1] = acc[ct][0][8 + bl * 4 + i];
              }
            }
            store8<F32>(reinterpret_cast<char*>(row + (blk * 32) % kPart + 16 * bl + 8 * g), x);
          }
        }
      if (g == 0) *reinterpret_cast<f32x4*>(row + kPart) = f32x4{m[ct], total, 0.f, 0.f};
      __syncthreads();
      for (int item = threadIdx.x; item < 32 * P; item += W * 64) {
        const int cc = item / P, d = item % P * 8, r = row0 + ct * 32 + cc;
        if (r >= rows) continue;
        const float* rec = reinterpret_cast<const float*>(s_mem) + cc * kRow;
        float M = kKv4Floor, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, rec[w * 32 * kRow + kPart]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float f = kv4_shift(rec[w * 32 * kRow + kPart], M, p.scale2);
          L = __builtin_fmaf(rec[w * 32 * kRow + kPart + 1], f, L);
          float y[8];
          load8<F32>(reinterpret_cast<const char*>(rec + w * 32 * kRow + d), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf(y[e], f, o[e]);
        }
        const int tok = r / p.G, hq = h * p.G + r % p.G;
        const int64_t orow = (int64_t)(q0 + tok) * p.Hq + hq;
        if (p.nsplit > 1) {
          float* out = p.ws + (orow * p.nsplit + sp) * (D + 4);
          store8<F32>(reinterpret_cast<char*>(out + part * kPart + d), o);
          if (d == 0 && part == 0) *reinterpret_cast<f32x4*>(out + D) = f32x4{M, L, 0.f, 0.f};
        } else {
          const bool any = limit(r) >= 0;
          const float inv = any ? 1.f / L : 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = any ? o[e] * inv : 0.f;
          store8<Tag>(p.out + (orow * D + part * kPart + d) * EB, o);
        }
      }
    }
  }
}

// Joins the splits of the segments' query rows; items are (segment, token, query head).
template <class Tag, int D, int SL>
__global__ void __launch_bounds__(256) kv4_prefill_merge_kernel(const Kv4PrefillParams p, int64_t items) {
  const int64_t item = (int64_t)blockIdx.x * (256 / (SL * D / 8)) + (SL == 1 ? threadIdx.x / (D / 8) : 0);
  if (item >= items) return;
  const int hq = (int)(item % p.Hq);
  const int64_t st = item / p.Hq;
  const int tok = (int)(st % p.max_q_len), seg = (int)(st / p.max_q_len);
  const int q0 = p.seg_q0[seg];
  if (tok >= segment_rows(p, q0, p.seg_len[seg])) return;
  const int lim = min(p.seg_pos0[seg] + tok, p.max_ctx - 1);
  const int64_t row = (int64_t)(q0 + tok) * p.Hq + hq;
  kv4_join_splits<Tag, D, SL>(p.out + row * D * Tag::kBytes, p.ws + row * p.nsplit * (D + 4),
                              lim < 0 ? 0 : min(lim / p.tps + 1, p.nsplit), p.scale2);
}
template <class Tag, int D, int SL>
void launch_merge(const Kv4PrefillParams& p, hipStream_t s) {
  const int64_t items = (int64_t)p.nseg * p.max_q_len * p.Hq;
  hipLaunchKernelGGL((kv4_prefill_merge_kernel<Tag, D, SL>), dim3((unsigned)ceil_div64(items, 256 / (SL * D / 8))), dim3(256), 0,
                     s, p, items);
}

struct Kv4PrefillPlan {
  bool dealt;            // kv4_rows_kernel, else kv4_prefill_kernel
  int tiles, waves, row_tiles;  // column tiles per wave, waves per workgroup; workgroups along a segment's rows
  int nsplit, tps;       // splits of the context, tokens of one
  size_t ws_bytes;
};

// Host arithmetic only.
int make_plan(const char* what, int nseg, int total_rows, int max_q_len, int Hq, int Hkv, int D, int max_ctx, int dtype,
              Kv4PrefillPlan* pl) {
  if (!kv4_dtype_ok(dtype)) return fail(MI355_EINVAL, "%s: dtype %d", what, dtype);
  if (!kv4_head_dim_ok(D)) return fail(MI355_EUNSUPPORTED, "%s: head_dim %d (the 4-bit cache holds 32, 64, 128 or 256)", what, D);
  if (nseg < 0 || total_rows < 0 || max_q_len < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || max_ctx <= 0 || max_ctx > kKv4MaxContext)
    return fail(MI355_EINVAL, "%s: bad shape (nseg=%d total_rows=%d max_q_len=%d Hq=%d Hkv=%d max_context=%d)", what, nseg,
                total_rows, max_q_len, Hq, Hkv, max_ctx);
  max_q_len = std::min(max_q_len, total_rows);
  const int64_t rows = (int64_t)max_q_len * (Hq / Hkv), heads = (int64_t)std::max(nseg, 1) * Hkv;
  if (rows > INT32_MAX) return fail(MI355_EINVAL, "%s: max_q_len %d", what, max_q_len);
  // kv4_rows_kernel has shorter walks and no barriers, but converts every code once per 32 (two tiles: 64) rows, where
  // kv4_prefill_kernel does per 64 (128): the former while its workgroups fit the chip about at once -- three of one tile per
  // CU, two beyond 64 dims; two of two tiles -- the latter beyond.  us, as chosen / the next best:
  //   dealt, one tile   8 chunks to 45 behind 900, 8 heads of 64 10.3 / 15.4; a prompt of 2000, 8 of 64 18 / 25; one of 500,
  //                     32/8 of 128 12.2 / 15.5; 2 of 128 behind 2000, 32/8 of 256 35 / 86; 5 of 512 behind 2000, 8 of 64, fp32
  //                     47 / 58; 2 of 200 .. 300 behind 500 .. 1500, 32/8 of 128, fp16 46 / 60
  //   dealt, two tiles  8 of 512 behind 2000, 8 of 64 43.0 / 43.3; 4 of 256 behind 3000, 32/8 of 128 82 / 89; a prompt of 2000,
  //                     32/8 of 128 62 / 68
  //   shared, one tile  16 uneven chunks to 1024, 8 of 64 34 / 33; 12 uneven fp16 prompts to 1500, 8 of 64 48.6 / 52.8; 3 of
  //                     256, 32/8 of 128 13.1 / 15.0; 16 of 500, fp16, 8 of 256 53 / 69
  //   shared, two tiles 8 of 4096, 8 of 64 234 / 250; 4 of 2048 behind 2048, 32/8 of 128 561 / 562; 8 of 1024, 8 of 128 43.0 / 42.6
  // Registers set limits: two tiles spill at head_dim 256 and fp32's 128, and fp16's 128 where they are dealt.
  const bool narrow = D == 256 || (dtype == MI355_F32 && D == 128), single = narrow || (dtype == MI355_F16 && D == 128);
  const int64_t all_rows = (int64_t)total_rows * (Hq / Hkv);
  auto workgroups = [&](int64_t per) {   // of uneven segments: no more than the rows there are
    return std::min(heads * ceil_div64(rows, per), Hkv * (ceil_div64(all_rows, per) + nseg));
  };
  const int64_t wgs = workgroups(32);
  pl->dealt = true;
  pl->tiles = 1;
  if (wgs > (single && max_ctx >= 768 ? 1024 : D <= 64 ? 768 : 512)) {
    pl->tiles = 2;
    if (single || max_ctx < 512 || workgroups(64) >= (D <= 64 ? 513 : 1024)) {
      pl->dealt = false;
      pl->tiles = !narrow && workgroups(128) > (D <= 64 ? 1023 : 256) ? 2 : 1;
    }
  }
  if (const int form = knob(kKnobKv4ChunkForm); form == 1 || form == 2 || form == 11 || form == 12) {
    pl->dealt = form > 10;
    pl->tiles = form % 10 == 2 && !(pl->dealt ? single : narrow) ? 2 : 1;
  }
  pl->row_tiles = (int)ceil_div64(rows, (pl->dealt ? 32 : 64) * pl->tiles);
  // Fewer workgroups than CUs: the context is split until there is one each, no split shorter than 256 tokens (16 tokens
  // behind 30000, 32/8 heads of 128: 169 -> 27 us; 4 chunks to 64 behind 1500, 8/2 heads of 256: 24.6 -> 21.0), if that takes
  // 1100 tokens off a walk: the merge costs a launch (4.4 us of the host's time where steps are not replayed) and the rows'
  // partial sums (2 chunks of 64 behind 2000, 32/8 heads of 128, replayed: 19.3 in one, 20.0 in two, 26.6 in four).
  // One workgroup per CU or fewer: eight waves each, if the walk is long enough to pay for the larger join (2 of 512 behind
  // 2000, 8 heads of 64, fp32 23.3 -> 21.4 us; 4 of 100 .. 200 behind 1500 .. 3000, 8 of 128 29.4 -> 25.8; 4 to 64 behind 600,
  // 8 of 64 9.4 and 9.2; 4 of 250, 8 of 64 7.0 and 7.3).
  pl->waves = pl->dealt && pl->tiles == 1 && wgs <= 256 && max_ctx >= 768 ? 8 : kWaves;
  const int stage = pl->waves * kKv4Step;
  const int64_t stages = ceil_div64(max_ctx, stage);
  int64_t want = pl->dealt && wgs <= 128 ? std::min<int64_t>(256 / std::max<int64_t>(wgs, 1), ceil_div64(max_ctx, 256)) : 1;
  if (max_ctx - max_ctx / want < 1100) want = 1;
  const int64_t per = ceil_div64(stages, std::min(want, stages));
  pl->tps = (int)(per * stage);
  pl->nsplit = (int)ceil_div64(stages, per);
  pl->ws_bytes = pl->nsplit > 1 ? (size_t)total_rows * Hq * pl->nsplit * (D + 4) * sizeof(float) : 0;
  if (!kv4_grid_ok(heads * pl->row_tiles * pl->nsplit, 64 * pl->waves) ||
      (pl->nsplit > 1 && !kv4_grid_ok((int64_t)nseg * max_q_len * Hq, 256)))
    return fail(MI355_EINVAL, "%s: too many workgroups (nseg=%d max_q_len=%d Hq=%d)", what, nseg, max_q_len, Hq);
  return 0;
}

template <class Tag, int D>
int launch(const Kv4PrefillParams& p, const Kv4PrefillPlan& pl, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.row_tiles * p.nseg * p.Hkv * p.nsplit)), block(256);
  constexpr bool narrow = D == 256 || (Tag::kBytes == 4 && D == 128), single = narrow || (Tag::kCode == MI355_F16 && D == 128);
  if (pl.tiles == 1) {
    if (pl.dealt && pl.waves == 8) hipLaunchKernelGGL((kv4_rows_kernel<Tag, D, 1, 8>), grid, dim3(512), 0, s, p);
    else if (pl.dealt) hipLaunchKernelGGL((kv4_rows_kernel<Tag, D, 1, kWaves>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((kv4_prefill_kernel<Tag, D, 16>), grid, block, 0, s, p);
  } else if (pl.dealt) {
    if constexpr (!single) hipLaunchKernelGGL((kv4_rows_kernel<Tag, D, 2, kWaves>), grid, block, 0, s, p);
  } else {
    if constexpr (!narrow) hipLaunchKernelGGL((kv4_prefill_kernel<Tag, D, 32>), grid, block, 0, s, p);
  }
  if (int rc = check_launch("kv4_prefill_kernel")) return rc;
  if (p.nsplit > 1) {
    if (p.nsplit <= kKv4WalkedSplits) launch_merge<Tag, D, kv4_split_lanes<D>(true)>(p, s);
    else launch_merge<Tag, D, kv4_split_lanes<D>(false)>(p, s);
    return check_launch("kv4_prefill_merge_kernel");
  }
  return 0;
}
template <class Tag>
int launch(const Kv4PrefillParams& p, const Kv4PrefillPlan& pl, int D, hipStream_t s) {
  switch (D) {
    case 32: return launch<Tag, 32>(p, pl, s);
    case 64: return launch<Tag, 64>(p, pl, s);
    case 128: return launch<Tag, 128>(p, pl, s);
    default: return launch<Tag, 256>(p, pl, s);
  }
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" size_t mi355_paged_prefill_kv4_workspace_bytes(int32_t nseg, int32_t total_rows, int32_t max_q_len,
                                                          int32_t Hq, int32_t Hkv, int32_t D, int32_t max_context,
                                                          int32_t dtype) {
  Kv4PrefillPlan pl;
  if (nseg == 0 || max_q_len == 0 || total_rows == 0) return 0;
  if (make_plan("paged_prefill_kv4", nseg, total_rows, max_q_len, Hq, Hkv, D, max_context, dtype, &pl)) return 0;
  return pl.ws_bytes;
}

extern "C" int mi355_paged_prefill_kv4(void* out, const void* q, int64_t q_stride_tok, const void* k_cache,
                                       const void* v_cache, const int32_t* block_tables, const int32_t* seg_q_start,
                                       const int32_t* seg_len, const int32_t* seg_pos0, int32_t nseg,
                                       int32_t total_rows, int32_t max_q_len, int32_t Hq, int32_t Hkv, int32_t D,
                                       int32_t block_size, int32_t max_blocks, int32_t num_blocks,
                                       int32_t max_context, int64_t stride_block, int64_t stride_head, float scale,
                                       int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (nseg == 0 || max_q_len == 0 || total_rows == 0) return 0;
  if (!out || !q || !block_tables || !seg_q_start || !seg_len || !seg_pos0)
    return fail(MI355_EINVAL, "paged_prefill_kv4: null pointer argument");
  if (int rc = kv4_check_cache("paged_prefill_kv4", k_cache, v_cache, Hkv, D, block_size, num_blocks, stride_block, stride_head))
    return rc;
  if (max_blocks <= 0) return fail(MI355_EINVAL, "paged_prefill_kv4: max_blocks %d", max_blocks);
  if ((int64_t)max_context > (int64_t)max_blocks * block_size) max_context = max_blocks * block_size;
  Kv4PrefillPlan pl;
  if (int rc = make_plan("paged_prefill_kv4", nseg, total_rows, max_q_len, Hq, Hkv, D, max_context, dtype, &pl)) return rc;
  const int epl = dtype == MI355_F32 ? 4 : 8;
  if (q_stride_tok % epl || q_stride_tok < (int64_t)Hq * D || (((uintptr_t)q | (uintptr_t)out) & 15))
    return fail(MI355_EINVAL, "paged_prefill_kv4: query rows must be 16-byte aligned and a token's heads packed");
  if (!kv4_out_ok(out, q, q_stride_tok, (int64_t)Hq * D, total_rows, dtype))
    return fail(MI355_EINVAL, "paged_prefill_kv4: the output overlaps the query rows without being them");
  if (pl.ws_bytes && (!workspace || workspace_bytes < pl.ws_bytes || ((uintptr_t)workspace & 15)))
    return fail(MI355_EWORKSPACE, "paged_prefill_kv4: workspace of %zu bytes needed (16-byte aligned), %zu given", pl.ws_bytes,
                workspace ? workspace_bytes : (size_t)0);
  Kv4PrefillParams p;
  p.out = static_cast<char*>(out);
  p.q = static_cast<const char*>(q);
  p.cache = kv4_cache(k_cache, v_cache, stride_block, stride_head, num_blocks, block_size / kKv4Tile);
  p.bt = block_tables;
  p.seg_q0 = seg_q_start;
  p.seg_len = seg_len;
  p.seg_pos0 = seg_pos0;
  p.q_stride = q_stride_tok;
  p.nseg = nseg;
  p.total_rows = total_rows;
  p.max_q_len = std::min(max_q_len, total_rows);
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.max_blocks = max_blocks;
  p.max_ctx = max_context;
  p.row_tiles = pl.row_tiles;
  p.nsplit = pl.nsplit;
  p.tps = pl.tps;
  p.ws = static_cast<float*>(workspace);
  p.flip = scale < 0.f;
  p.scale2 = std::max(std::fabs(scale) * 1.44269504088896340736f, 1e-30f);   // (a scale of 0: all weights 1 to 30 digits)
  p.raise = kKv4Raise / p.scale2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MI355_F32: return launch<F32>(p, pl, D, s);
    case MI355_BF16: return launch<BF16>(p, pl, D, s);
    default: return launch<F16>(p, pl, D, s);
  }
}
