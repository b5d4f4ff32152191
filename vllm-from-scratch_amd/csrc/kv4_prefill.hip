// Attention of several new query tokens per sequence over the 4-bit KV cache (their K / V rows are in
// it already): query j of a segment attends to positions 0 .. pos0 + j.
//
// The query rows of a (segment, kv head) are its (token, query head of the group) pairs.  A workgroup
// of four waves owns 4 x MC tiles of 16 of them (a tile is the 16 columns of a score tile) and walks the
// context in stages of SUB steps of 32 tokens.  Per stage each wave converts a quarter of the K and V
// codes to bf16 (exact) and leaves them in LDS as the operands of the matrix instruction; every wave
// reads them all back, once per MC tiles.  Conversion is what the format costs beside attention in
// bf16: 130 vector instructions per 32 tokens of 128 dims, as many as two tiles' softmax, so it is done
// once per workgroup and not once per wave.  Codes travel from memory one stage ahead in registers,
// operands one stage ahead in LDS (two buffers, one barrier per stage).
// A stage is a chain -- scores, softmax, values, barrier -- that eight waves of a CU overlap and four do not.
// Where there are few workgroups each gets a second team of four waves for the same rows; the teams take
// the stages in turn and are joined through LDS.
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

template <class Tag, int D, int MC, int TEAMS>
__global__ void __launch_bounds__(256 * TEAMS, 2) kv4_prefill_kernel(const Kv4PrefillParams p) {
  typedef Stage<D> St;
  constexpr int NP = Kv4Pieces<Tag>::n, KS = D / 32, EB = Tag::kBytes, SUB = St::SUB, NB = St::NB, KT = St::KT, KF = St::KF;
  constexpr int KA = KS < 4 ? KS : 4, VA = KS < 2 ? KS : 2;   // operands read ahead of their use
  struct Shared {   // one team's
    bf16x8_t k[2][SUB][2][KS][64], v[2][SUB][KS][2][64];
    uint32_t nan[2][SUB][KS];   // tokens of a step whose V block was NaN (masked stages only)
  };
  constexpr int kRow = D + 4;   // a column's sums, maximum and sum of weights on their way from team 1 to team 0
  constexpr int kShared = TEAMS * (int)sizeof(Shared), kJoin = TEAMS > 1 ? kWaves * MC * 16 * kRow * 4 : 0;
  __shared__ __attribute__((aligned(16))) char s_mem[kShared > kJoin ? kShared : kJoin];
  const int lane = threadIdx.x & 63, wg_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = TEAMS > 1 ? wg_wave / kWaves : 0, wave = TEAMS > 1 ? wg_wave % kWaves : wg_wave;
  Shared& sh = reinterpret_cast<Shared*>(s_mem)[team];
  const int g = lane >> 4, col = lane & 15;
  int idx = blockIdx.x;
  const int sp = idx % p.nsplit;
  idx /= p.nsplit;
  const int h = idx % p.Hkv;   // (kv heads on neighbouring XCDs: the row tiles of one head share an L2 where Hkv is a multiple of 8)
  idx /= p.Hkv;
  const int seg = idx % p.nseg;
  const int rt = p.row_tiles - 1 - idx / p.nseg;   // the longest contexts first
  const int q0 = p.seg_q0[seg], pos0 = p.seg_pos0[seg], len = segment_rows(p, q0, p.seg_len[seg]);
  const int rows = len * p.G, wg_row0 = rt * kWaves * MC * 16;
  if (wg_row0 >= rows) return;
  const int row0 = wg_row0 + wave * MC * 16;

  int lim[MC];       // last position the column attends to; -1: none
  int64_t orow[MC];  // its row of out (and of q), -1: none
  bf16x8_t qf[MC][KS][NP];
#pragma unroll
  for (int mc = 0; mc < MC; ++mc) {
    const int r = row0 + mc * 16 + col, rr = min(r, rows - 1);
    const int tok = rr / p.G, hq = h * p.G + rr % p.G;
    lim[mc] = min(pos0 + tok, p.max_ctx - 1);
    orow[mc] = r < rows ? (int64_t)(q0 + tok) * p.Hq + hq : -1;
    const char* src = p.q + ((int64_t)(q0 + tok) * p.q_stride + (int64_t)hq * D + g * (D / 4)) * EB;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
      load8<Tag>(src + s * 8 * EB, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = p.flip ? -x[e] : x[e];
      bf16_pieces<NP>(x, qf[mc][s]);
    }
  }
  auto limit = [&](int r) { return min(pos0 + min(r, rows - 1) / p.G, p.max_ctx - 1); };
  const int wave_first = limit(row0);
  const int wg_first = limit(wg_row0), wg_end = limit(wg_row0 + kWaves * MC * 16 - 1);
  const int lo = sp * p.tps, wg_last = min(wg_end, lo + p.tps - 1);   // this workgroup's tokens: lo .. wg_last
  const int wave_last = row0 < rows ? min(limit(row0 + MC * 16 - 1), wg_last) : -1;
  if (lo > wg_last && sp > 0) return;                                 // (the rows' own limits tell which splits are empty)

  f32x4 acc[MC][KS][2], sum[MC];
  float m[MC], m2[MC];   // running maximum of the raw scores, and times the scale
#pragma unroll
  for (int mc = 0; mc < MC; ++mc) {
    m[mc] = m2[mc] = kKv4Floor;
    sum[mc] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) acc[mc][s][0] = acc[mc][s][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bf16x8_t ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (__bf16)1.f;

  // ---- this wave's part of a stage
  const int32_t* table = p.bt + (int64_t)seg * p.max_blocks;
  const int last_tile = max(wg_last, 0) / kKv4Tile;
  const int vstep = St::step(wave), vblk = St::v_block(wave), kstep = vstep, ktile = St::k_tile(wave),
            kfirst = St::k_first(wave);
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
      // for the columns that see them, where the stage is used.
      uint32_t nan[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) nan[b] = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int live = wg_last + 1 - (t0 + vstep * kKv4Step + i * kKv4Tile + 4 * g);   // of this lane's four tokens
        const uint32_t keep = live >= 4 ? ~0u : (live <= 0 ? 0u : (1u << (8 * live)) - 1u);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t vs = (rvs[i][b] & keep) | (0x7f7f7f7fu & ~keep), bad = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool is_nan = ((vs >> (8 * j)) & 0xffu) == 255u;
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
        for (int b = 0; b < NB; ++b) sh.nan[buf][vstep][vblk + b] = nan[b];
      }
    }
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const float sc = u2f(__builtin_amdgcn_alignbit(rks[i], rks[i], turn));
#pragma unroll
      for (int f = 0; f < KF; ++f) sh.k[buf][kstep][KT == 2 ? i : ktile][kfirst + f][lane] = kv4_k_frag(rk[i][f], sc);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      bf16x8_t ev, od;
      kv4_v_frags(rv[0][b], rv[1][b], rvs[0][b], rvs[1][b], ev, od);
      sh.v[buf][vstep][vblk + b][0][lane] = ev;
      sh.v[buf][vstep][vblk + b][1][lane] = od;
    }
  };

  if (wg_last >= lo) {
    constexpr int kStride = TEAMS * St::kTokens;   // the teams take stages in turn
    const int first = lo + team * St::kTokens;
    place(first);
    fetch();
    place(first + kStride);
    convert(first, 0);
    fetch();
    place(first + 2 * kStride);
    int buf = 0;
    for (int t0 = first; t0 - team * St::kTokens <= wg_last; t0 += kStride, buf ^= 1) {
      lds_barrier();
      convert(t0 + kStride, buf ^ 1);   // (behind the last stage: the last tile again, read by nobody)
      fetch();
      place(min(t0 + 3 * kStride, wg_last));
      const bool wg_masked = t0 + St::kTokens - 1 > wg_first;
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        const int ts = t0 + sub * kKv4Step;
        if (ts > wave_last) break;
        const bool masked = ts + kKv4Step - 1 > wave_first;
        f32x4 S[MC][2];
        bf16x8_t kf[2][KA];   // K operands, read 2 KA ahead
#pragma unroll
        for (int f = 0; f < 2 * KA; ++f) kf[f / KA][f % KA] = sh.k[buf][sub][f / KS][f % KS][lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int mc = 0; mc < MC; ++mc) S[mc][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int f = i * KS + s;
            const bf16x8_t a = kf[f / KA % 2][f % KA];
            if (f + 2 * KA < 2 * KS) kf[f / KA % 2][f % KA] = sh.k[buf][sub][(f + 2 * KA) / KS][(f + 2 * KA) % KS][lane];
#pragma unroll
            for (int mc = 0; mc < MC; ++mc)
#pragma unroll
              for (int n = 0; n < NP; ++n) S[mc][i] = mfma_bf16(a, qf[mc][s][n], S[mc][i]);
          }
        }
        bf16x8_t vf[VA][2];   // V operands of the first blocks, on their way during the softmax
#pragma unroll
        for (int s = 0; s < VA; ++s) {
          vf[s][0] = sh.v[buf][sub][s][0][lane];
          vf[s][1] = sh.v[buf][sub][s][1][lane];
        }
        __builtin_amdgcn_sched_barrier(0);
        if (wg_masked) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const uint32_t nan = __builtin_amdgcn_readfirstlane(sh.nan[buf][sub][s]);
            if (nan) {
#pragma unroll
              for (int mc = 0; mc < MC; ++mc) {
                const int seen = lim[mc] + 1 - ts;   // tokens of the step the column sees
                const uint32_t sees = seen >= 32 ? ~0u : (seen <= 0 ? 0u : (1u << seen) - 1u);
                if (nan & sees) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[mc][s][0][e] = acc[mc][s][1][e] = __builtin_nanf("");
                }
              }
            }
          }
        }
        bf16x8_t pf[MC][NP];
#pragma unroll
        for (int mc = 0; mc < MC; ++mc) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = S[mc][e >> 2][e & 3];
          if (masked) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (ts + (e >> 2) * kKv4Tile + 4 * g + (e & 3) > lim[mc]) x[e] = -INFINITY;
          }
          float top = fmaxf(fmaxf(x[0], x[1]), x[2]);
          top = fmaxf(fmaxf(top, x[3]), x[4]);
          top = fmaxf(fmaxf(top, x[5]), fmaxf(x[6], x[7]));
          if (__ballot(top > m[mc] + p.raise)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = fmaxf(m[mc], top), f = fast_exp2((m[mc] - mn) * p.scale2);
            m[mc] = mn;
            m2[mc] = fmaxf(mn * p.scale2, kKv4Floor);
            sum[mc] *= f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              acc[mc][s][0] *= f;
              acc[mc][s][1] *= f;
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = fast_exp2(__builtin_fmaf(x[e], p.scale2, -m2[mc]));
          bf16_pieces<NP>(x, pf[mc]);
#pragma unroll
          for (int n = 0; n < NP; ++n) sum[mc] = mfma_bf16(ones, pf[mc][n], sum[mc]);   // every row: the column's sum of weights
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const bf16x8_t ev = vf[s % VA][0], od = vf[s % VA][1];
          if (s + VA < KS) {
            vf[s % VA][0] = sh.v[buf][sub][s + VA][0][lane];
            vf[s % VA][1] = sh.v[buf][sub][s + VA][1][lane];
          }
#pragma unroll
          for (int mc = 0; mc < MC; ++mc)
#pragma unroll
            for (int n = 0; n < NP; ++n) {
              acc[mc][s][0] = mfma_bf16(ev, pf[mc][n], acc[mc][s][0]);
              acc[mc][s][1] = mfma_bf16(od, pf[mc][n], acc[mc][s][1]);
            }
        }
      }
    }
  }

  if constexpr (TEAMS > 1) {
    float* const join = reinterpret_cast<float*>(s_mem) + (wave * MC * 16 + col) * kRow;
    __syncthreads();   // (nobody reads operands any more)
    if (team == 1) {
#pragma unroll
      for (int mc = 0; mc < MC; ++mc) {
        float* const row = join + mc * 16 * kRow;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          *reinterpret_cast<f32x4*>(row + 32 * s + 8 * g) = acc[mc][s][0];
          *reinterpret_cast<f32x4*>(row + 32 * s + 8 * g + 4) = acc[mc][s][1];
        }
        if (g == 0) row[D] = m2[mc], row[D + 1] = sum[mc][0];
      }
    }
    __syncthreads();
    if (team == 1) return;
#pragma unroll
    for (int mc = 0; mc < MC; ++mc) {
      const float* const row = join + mc * 16 * kRow;
      const float M = fmaxf(m2[mc], row[D]), fa = fast_exp2(m2[mc] - M), fb = fast_exp2(row[D] - M);
      m2[mc] = M;
      sum[mc][0] = __builtin_fmaf(row[D + 1], fb, sum[mc][0] * fa);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const f32x4 e = *reinterpret_cast<const f32x4*>(row + 32 * s + 8 * g), o = *reinterpret_cast<const f32x4*>(row + 32 * s + 8 * g + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[mc][s][0][i] = __builtin_fmaf(e[i], fb, acc[mc][s][0][i] * fa);
          acc[mc][s][1][i] = __builtin_fmaf(o[i], fb, acc[mc][s][1][i] * fa);
        }
      }
    }
  }
#pragma unroll
  for (int mc = 0; mc < MC; ++mc) {
    if (orow[mc] < 0) continue;
    if (p.nsplit > 1) {
      float* rec = p.ws + (orow[mc] * p.nsplit + sp) * (D + 4);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const f32x4 e = acc[mc][s][0], o = acc[mc][s][1];
        *reinterpret_cast<f32x4*>(rec + 32 * s + 8 * g) = f32x4{e[0], o[0], e[1], o[1]};
        *reinterpret_cast<f32x4*>(rec + 32 * s + 8 * g + 4) = f32x4{e[2], o[2], e[3], o[3]};
      }
      if (g == 0) *reinterpret_cast<f32x4*>(rec + D) = f32x4{m2[mc], sum[mc][0], 0.f, 0.f};
      continue;
    }
    const float inv = lim[mc] >= 0 ? 1.f / sum[mc][0] : 0.f;   // a query before position 0 sees nothing: zeros
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const f32x4 e = acc[mc][s][0], o = acc[mc][s][1];
      float x[8] = {e[0], o[0], e[1], o[1], e[2], o[2], e[3], o[3]};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = lim[mc] >= 0 ? x[i] * inv : 0.f;
      store8<Tag>(p.out + (orow[mc] * D + 32 * s + 8 * g) * EB, x);
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
                              lim < 0 ? 0 : min(lim / p.tps + 1, p.nsplit));
}
template <class Tag, int D, int SL>
void launch_merge(const Kv4PrefillParams& p, hipStream_t s) {
  const int64_t items = (int64_t)p.nseg * p.max_q_len * p.Hq;
  hipLaunchKernelGGL((kv4_prefill_merge_kernel<Tag, D, SL>), dim3((unsigned)ceil_div64(items, 256 / (SL * D / 8))), dim3(256), 0,
                     s, p, items);
}

struct Kv4PrefillPlan {
  int MC, teams, row_tiles, nsplit, tps;
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
  // Two tiles of 16 rows per wave use every converted operand twice, one tile makes twice the workgroups.  Two teams per
  // workgroup halve the stages of its walk and fill a chip that has too few workgroups, but take twice its LDS: they pay while
  // all workgroups fit at once, one per CU, or (deep contexts, up to 64 dims) two.  us, as chosen / the other way:
  //   two tiles: 8 prompts of 4096, 8 heads of 64 172 / 197; 8 of 1024, 8 of 128 37 / 42; 4 of 300, 32/8 of 128 32 / 37
  //   one tile: 16 uneven chunks to 1024, 8 of 64 43 / 47; 12 uneven fp16 prompts to 1500 49 / 54; 5 of 512, 8 of 128 17 / 22
  //   two teams: a prompt of 2000, 8 heads of 64 22 / 29; one of 500, 32/8 of 128 14.4 / 16.3; 2 of 128 behind 2000, 32/8 of
  //   256 44 / 78; 8 of 512 behind 2000, 8 of 64 38 / 46; two tiles: 4 of 256 behind 3000, 32/8 of 128 67 / 88
  //   one team: 12 uneven prompts to 400, 8 of 64 10.7 / 12.2; 8 of 4096, 8 of 64 172 / 228; 16 of 100 7.5 / 7.9
  // Two tiles' registers at head_dim 256 (fp32: 128) would leave one wave per SIMD.
  const bool narrow = D == 256 || (dtype == MI355_F32 && D == 128);
  const int64_t all_rows = (int64_t)total_rows * (Hq / Hkv);
  auto workgroups = [&](int mc) {   // of uneven segments: no more than the rows there are
    const int64_t per = kWaves * 16 * mc;
    return std::min(heads * ceil_div64(rows, per), Hkv * (ceil_div64(all_rows, per) + nseg));
  };
  const int64_t wgs1 = workgroups(1), wgs2 = workgroups(2);
  const bool deep = max_ctx >= 1536;
  pl->MC = !narrow && (D <= 64 ? wgs2 >= 1024 : wgs2 > 256 || (wgs1 > 256 && deep)) ? 2 : 1;
  pl->teams = 1;
  if (max_ctx >= 256 && wgs1 <= 256) pl->teams = 2;
  if (deep && (D <= 64 ? wgs1 <= 512 : pl->MC == 2 && wgs2 <= 256)) pl->teams = 2;
  pl->row_tiles = (int)ceil_div64(rows, kWaves * pl->MC * 16);
  const int stage = kKv4Step * (D == 256 ? 1 : D == 32 ? 4 : 2);
  const int64_t stages = ceil_div64(max_ctx, stage);
  // Still fewer than one workgroup per CU: the context is split until there is one, no split shorter than 256 tokens (16
  // tokens behind 30000, 32/8 heads of 128: 348 -> 27 us; 8 chunks to 64 behind 2000, 8 heads of 64: 23.2 -> 15.4), if that
  // takes 800 tokens off a walk.  The merge costs a launch (4.4 us of the host's time) and the rows' partial sums: 8 chunks
  // to 45 behind 900 take 13.9 in one, 12.4 in four splits and 17 where the host is what they wait for; 128 tokens behind
  // 1000, 32/8 heads of 128, 21.5 in one, 22.9 in two.
  int64_t want = wgs1 <= 256 ? std::min<int64_t>(256 / std::max<int64_t>(wgs1, 1), ceil_div64(max_ctx, 256)) : 1;
  if (max_ctx - max_ctx / want < 800) want = 1;
  const int64_t per = ceil_div64(stages, std::min(want, stages));
  pl->tps = (int)(per * stage);
  pl->nsplit = (int)ceil_div64(stages, per);
  pl->ws_bytes = pl->nsplit > 1 ? (size_t)total_rows * Hq * pl->nsplit * (D + 4) * sizeof(float) : 0;
  if (!kv4_grid_ok(heads * pl->row_tiles * pl->nsplit, 256 * pl->teams) ||
      (pl->nsplit > 1 && !kv4_grid_ok((int64_t)nseg * max_q_len * Hq, 256)))
    return fail(MI355_EINVAL, "%s: too many workgroups (nseg=%d max_q_len=%d Hq=%d)", what, nseg, max_q_len, Hq);
  return 0;
}

template <class Tag, int D>
int launch(const Kv4PrefillParams& p, const Kv4PrefillPlan& pl, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.row_tiles * p.nseg * p.Hkv * p.nsplit)), one(256), two(512);
  if constexpr (D < 256 && !(Tag::kCode == MI355_F32 && D == 128)) {
    if (pl.MC == 2 && pl.teams == 1) hipLaunchKernelGGL((kv4_prefill_kernel<Tag, D, 2, 1>), grid, one, 0, s, p);
    if constexpr (D == 128)
      if (pl.MC == 2 && pl.teams == 2) hipLaunchKernelGGL((kv4_prefill_kernel<Tag, D, 2, 2>), grid, two, 0, s, p);
  }
  if (pl.MC == 1 && pl.teams == 1) hipLaunchKernelGGL((kv4_prefill_kernel<Tag, D, 1, 1>), grid, one, 0, s, p);
  if (pl.MC == 1 && pl.teams == 2) hipLaunchKernelGGL((kv4_prefill_kernel<Tag, D, 1, 2>), grid, two, 0, s, p);
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
