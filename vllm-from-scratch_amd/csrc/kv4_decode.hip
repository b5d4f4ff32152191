// Decode attention (one query token per sequence) over the 4-bit KV cache.
//
// A wave owns up to 16 query heads -- the 16 columns of a score tile -- that read NH neighbouring
// kv heads, and walks its tokens in steps of 32 (two cache tiles).  Per step and kv head the K tiles
// are converted to bf16 (exact) and multiplied with the queries of ALL columns; a column keeps the
// product of its own kv head, so that the softmax of a step runs once on a full tile whatever the
// number of query heads per kv head.  The weights go back into the matrix unit in the registers they
// were born in (see kv4.h) against the same step's V tiles; every kv head accumulates into registers
// of its own, so a NaN in one head never meets another.  The running maximum is only raised when a
// score passes it by more than kKv4Raise powers of two: until then the sums stay on the old one.
// The waves of a workgroup take steps in turn and combine their sums in LDS; a long context is
// split over workgroups, whose partial sums kv4_merge_kernel joins.
#include <algorithm>
#include <cmath>

#include "kv4.h"

namespace mi355 {
namespace {

struct Kv4DecodeParams {
  char* out;
  const char* q;
  Kv4Cache cache;
  const int32_t* bt;
  const int32_t* ctx;
  float* ws;   // [B * Hq][nsplit][D + 4]: unnormalised sums, running maximum, sum of weights
  int64_t q_stride;   // elements
  int B, Hq, Hkv, G /* query heads per kv head */, gc /* of them per workgroup */, qchunks, hgroups;
  int max_blocks, max_ctx, nsplit, tps /* tokens per split */;
  float scale2, raise;   // |scale| * log2(e); kKv4Raise in units of a raw score
  int flip;              // a negative scale: the queries are negated
};

template <class Tag, int D, int NH, int W>
__global__ void __launch_bounds__(W * 64) kv4_decode_kernel(const Kv4DecodeParams p) {
  constexpr int NP = Kv4Pieces<Tag>::n, NW = Kv4Pieces<Tag>::weights, KS = D / 32, EB = Tag::kBytes;
  __shared__ float s_o[W][16][D + 4];
  __shared__ float s_m[W][16], s_l[W][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  Kv4Lane<D> at(lane);
  int idx = blockIdx.x;
  const int sp = idx % p.nsplit;
  idx /= p.nsplit;
  const int qc = idx % p.qchunks;
  idx /= p.qchunks;
  const int hg = idx % p.hgroups, b = idx / p.hgroups;
  const int h0 = hg * NH;
  // column -> (kv head h0 + my_j, query head of its group)
  const int my_j = col / p.gc, my_q = qc * p.gc + col % p.gc;
  const bool used = my_j < NH && my_q < p.G;
  const int hq = (h0 + my_j) * p.G + my_q;

  const int ctx = min(p.ctx[b], p.max_ctx);
  const int lo = sp * p.tps, hi = min(ctx, lo + p.tps);   // this workgroup's tokens
  if (lo >= hi && p.nsplit > 1) return;                   // (the merge knows which splits are empty)

  bf16x8_t qf[KS][NP];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (used) load8<Tag>(p.q + ((int64_t)b * p.q_stride + (int64_t)hq * D + g * (D / 4) + s * 8) * EB, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p.flip ? -x[e] : x[e];
    bf16_pieces<NP>(x, qf[s]);
  }
  f32x4 acc[NH][KS][2], sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NH; ++j)
#pragma unroll
    for (int s = 0; s < KS; ++s) acc[j][s][0] = acc[j][s][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kKv4Floor;   // running maximum of the raw scores
  bf16x8_t ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (__bf16)1.f;

  const int32_t* table = p.bt + (int64_t)b * p.max_blocks;
  const char* const kbase = p.cache.k + (int64_t)h0 * p.cache.s_head;
  const char* const vbase = p.cache.v + (int64_t)h0 * p.cache.s_head;
  const int last_tile = (hi - 1) / kKv4Tile;
  // (a step's second tile may lie beyond the context: the last one is read twice)
  auto place = [&](int t, int i) { return kv4_place(p.cache, table, min((int)((uint32_t)t / kKv4Tile) + i, last_tile)); };
  auto record = [&](Kv4Place at) { return kv4_record(p.cache, at, kv4_tile_bytes(D)); };
  Kv4TileRegs<D> T[NH][2];
  auto fetch_k = [&](int64_t r0, int64_t r1) {
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      kv4_load_k<D, true>(scalar_base(kbase + r0 + j * p.cache.s_head), at, T[j][0]);
      kv4_load_k<D, true>(scalar_base(kbase + r1 + j * p.cache.s_head), at, T[j][1]);
    }
  };
  auto fetch_v = [&](int64_t r0, int64_t r1) {
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      kv4_load_v<D, true>(scalar_base(vbase + r0 + j * p.cache.s_head), at, T[j][0]);
      kv4_load_v<D, true>(scalar_base(vbase + r1 + j * p.cache.s_head), at, T[j][1]);
    }
  };

  constexpr int kStride = W * kKv4Step;
  int t0 = lo + wave * kKv4Step;
  // the table entries of the next step, asked for a step ahead of the loads that need them: waiting for an
  // entry in front of its loads would put one more trip to memory into every step
  Kv4Place n0{}, n1{};
  if (t0 < hi) {
    const Kv4Place a0 = place(t0, 0), a1 = place(t0, 1);
    n0 = place(min(t0 + kStride, hi - 1), 0), n1 = place(min(t0 + kStride, hi - 1), 1);
    const int64_t r0 = record(a0), r1 = record(a1);
    fetch_k(r0, r1);
    fetch_v(r0, r1);
  }
  // K registers are refilled for the next step as soon as the scores are made, V registers as soon as the
  // weights have met them: each load has the other half of a step to arrive.  The last step refills them
  // with the tile it has just read: a branch around the loads would make the compiler wait for all of them.
  for (; t0 < hi; t0 += kStride) {
    f32x4 S[2];
#pragma unroll
    for (int j = 0; j < NH; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4 c = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const bf16x8_t a = kv4_k_frag(T[j][i].k[s], kv4_k_scale<D>(T[j][i], at, s));
#pragma unroll
          for (int n = 0; n < NP; ++n) c = mfma_bf16(a, qf[s][n], c);
        }
        if (j == 0) S[i] = c;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) S[i][e] = my_j == j ? c[e] : S[i][e];
      }
    }
    const int64_t r0 = record(n0), r1 = record(n1);
    fetch_k(r0, r1);
    const int after = min(t0 + 2 * kStride, hi - 1);
    n0 = place(after, 0), n1 = place(after, 1);
    float x[8];   // tokens 4 g + e of each tile
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = S[e >> 2][e & 3];
    if (t0 + kKv4Step > hi) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (t0 + (e >> 2) * kKv4Tile + 4 * g + (e & 3) >= hi) x[e] = -INFINITY;
      // rows behind the context hold whatever was there: their codes count as 0 and their scales as 1
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int live = hi - (t0 + i * kKv4Tile + 4 * g);   // of this lane's four tokens
        const uint32_t keep = live >= 4 ? ~0u : (live <= 0 ? 0u : (1u << (8 * live)) - 1u);
#pragma unroll
        for (int j = 0; j < NH; ++j)
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            T[j][i].v[s] &= keep;
            T[j][i].vs[s] = (T[j][i].vs[s] & keep) | (0x7f7f7f7fu & ~keep);
          }
      }
    }
    float top = fmaxf(fmaxf(x[0], x[1]), x[2]);
    top = fmaxf(fmaxf(top, x[3]), x[4]);
    top = fmaxf(fmaxf(top, x[5]), fmaxf(x[6], x[7]));
    if (__ballot(top > m + p.raise)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top), f = kv4_shift(m, mn, p.scale2);
      m = mn;
      sum *= f;
#pragma unroll
      for (int j = 0; j < NH; ++j)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          acc[j][s][0] *= f;
          acc[j][s][1] *= f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = kv4_weight(x[e], m, p.scale2);
    bf16x8_t pf[NW];
    weight_pieces<NW>(x, pf);
#pragma unroll
    for (int n = 0; n < NW; ++n) sum = mfma_bf16(ones, pf[n], sum);   // every row: the column's sum of weights
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf16x8_t ev, od;
        kv4_v_frags(T[j][0].v[s], T[j][1].v[s], T[j][0].vs[s], T[j][1].vs[s], ev, od);
#pragma unroll
        for (int n = 0; n < NW; ++n) {
          acc[j][s][0] = mfma_bf16(ev, pf[n], acc[j][s][0]);
          acc[j][s][1] = mfma_bf16(od, pf[n], acc[j][s][1]);
        }
      }
    fetch_v(r0, r1);
  }

  // the lane's column: dims 32 s + 8 g .. + 8 (even and odd rows of the two accumulators alternate)
  if (g == 0) {
    s_m[wave][col] = m;
    s_l[wave][col] = sum[0];
  }
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    f32x4 e = acc[0][s][0], o = acc[0][s][1];
#pragma unroll
    for (int j = 1; j < NH; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = my_j == j ? acc[j][s][0][i] : e[i];
        o[i] = my_j == j ? acc[j][s][1][i] : o[i];
      }
    }
    float* dst = &s_o[wave][col][32 * s + 8 * g];
    *reinterpret_cast<f32x4*>(dst) = f32x4{e[0], o[0], e[1], o[1]};
    *reinterpret_cast<f32x4*>(dst + 4) = f32x4{e[2], o[2], e[3], o[3]};
  }
  __syncthreads();
  // columns x pieces of eight dims over the workgroup's threads
  constexpr int P = D / 8;
  for (int item = threadIdx.x; item < 16 * P; item += W * 64) {
    const int c = item / P, d = (item % P) * 8;
    const int j = c / p.gc, qi = qc * p.gc + c % p.gc;
    if (j >= NH || qi >= p.G) continue;
    float M = s_m[0][c];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, s_m[w][c]);
    float L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = kv4_shift(s_m[w][c], M, p.scale2);
      L = __builtin_fmaf(s_l[w][c], f, L);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf(s_o[w][c][d + e], f, o[e]);
    }
    const int64_t row = (int64_t)b * p.Hq + (int64_t)(h0 + j) * p.G + qi;
    if (p.nsplit == 1) {
      const float inv = ctx > 0 ? 1.f / L : 0.f;   // no token at all: zeros
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = ctx > 0 ? o[e] * inv : 0.f;
      store8<Tag>(p.out + (row * D + d) * EB, o);
    } else {
      float* rec = p.ws + (row * p.nsplit + sp) * (D + 4);
      *reinterpret_cast<f32x4*>(rec + d) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(rec + d + 4) = f32x4{o[4], o[5], o[6], o[7]};
      if (d == 0) *reinterpret_cast<f32x4*>(rec + D) = f32x4{M, L, 0.f, 0.f};
    }
  }
}

template <class Tag, int D, int SL>
__global__ void __launch_bounds__(256)
kv4_merge_kernel(char* out, const float* ws, const int32_t* ctx_lens, int rows, int Hq, int max_ctx, int nsplit, int tps,
                 float scale2) {
  const int64_t row = (int64_t)blockIdx.x * (256 / (SL * D / 8)) + (SL == 1 ? threadIdx.x / (D / 8) : 0);
  if (row >= rows) return;
  const int ctx = min(ctx_lens[row / Hq], max_ctx);
  kv4_join_splits<Tag, D, SL>(out + row * D * Tag::kBytes, ws + row * nsplit * (D + 4),
                              ctx <= 0 ? 0 : min(nsplit, (ctx + tps - 1) / tps), scale2);
}
template <class Tag, int D, int SL>
void launch_merge(const Kv4DecodeParams& p, hipStream_t s) {
  const int rows = p.B * p.Hq;
  hipLaunchKernelGGL((kv4_merge_kernel<Tag, D, SL>), dim3((unsigned)ceil_div64(rows, 256 / (SL * D / 8))), dim3(256), 0, s,
                     p.out, p.ws, p.ctx, rows, p.Hq, p.max_ctx, p.nsplit, p.tps, p.scale2);
}

struct Kv4Plan {
  int NH, W, gc, qchunks, hgroups, nsplit, tps;
  size_t ws_bytes;
};

// Host arithmetic only.  Figures: us per call, 8 heads of 64 in bf16 unless said otherwise.
int make_plan(const char* what, int B, int Hq, int Hkv, int D, int max_ctx, int dtype, Kv4Plan* pl) {
  if (!kv4_dtype_ok(dtype)) return fail(MI355_EINVAL, "%s: dtype %d", what, dtype);
  if (!kv4_head_dim_ok(D)) return fail(MI355_EUNSUPPORTED, "%s: head_dim %d (the 4-bit cache holds 32, 64, 128 or 256)", what, D);
  if (B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || max_ctx < 0 || max_ctx > kKv4MaxContext)
    return fail(MI355_EINVAL, "%s: bad shape (B=%d Hq=%d Hkv=%d max_context=%d)", what, B, Hq, Hkv, max_ctx);
  const int G = Hq / Hkv;
  pl->gc = std::min(G, 16);
  pl->qchunks = (G + 15) / 16;
  // kv heads per wave: more of them share a step's softmax and read longer runs of a block, but make fewer, longer
  // workgroups.  Where there is one (sequence, kv head) per CU or more, as many as leave a workgroup per CU: 256 x 2048
  // 61.7 / 56.8 / 54.6 with 1 / 2 / 4 heads, 64 x 2048 20.2 / 18.4 / 21.8, 64 x 4096 at head_dim 32 30.2 / 21.1 / 23.6, 32 x 4000
  // at head_dim 128 28.1 / 30.6.  Below that the context is split all the same, and long ones (in `units` of a kv head's 128
  // tokens) make up for the longer steps: 8 x 30000 35.2 / 31.1 / 32.4, 16 x 4000 15.6 / 16.0 / 15.5, 16 x 16000 at head_dim
  // 32, fp32, 34.9 / 26.3 / 23.8, 4 to 65536, 32/8 heads of 128, fp16, 47.4 / 45.5.  The accumulators of NH heads take
  // NH D / 2 registers: NH D <= 256 leaves room for two waves per SIMD.
  const int64_t heads = (int64_t)std::max(B, 1) * Hkv * pl->qchunks, units = heads * (((int64_t)max_ctx + 127) / 128);
  auto more = [&](int nh) {   // whether 2 nh heads are better than nh
    return heads < 256 ? units >= (int64_t)128 * D * nh : heads / (2 * nh) >= 256 && units >= (int64_t)4096 * nh;
  };
  pl->NH = 1;
  while (pl->NH * 2 <= 256 / D && pl->NH * 2 * pl->gc <= 16 && Hkv % (pl->NH * 2) == 0 && more(pl->NH)) pl->NH *= 2;
  if (const int nh = knob(kKnobKv4DecodeHeads); nh > 0 && (nh & (nh - 1)) == 0 && nh <= 256 / D && nh * pl->gc <= 16 && Hkv % nh == 0) pl->NH = nh;
  pl->hgroups = Hkv / pl->NH;
  const int64_t groups = (int64_t)std::max(B, 1) * pl->hgroups * pl->qchunks;
  // More workgroups than the chip's 256 CUs: four waves each.  Fewer: eight waves each as long as that leaves a wave few
  // steps (1 x 500: 6.3, in two splits and their merge 7.6; 32 x 1000: 9.2 against 10.6 with four waves), else the context
  // is split over workgroups, two per CU (1 x 8000: 9.2, whole 29.0; 8 x 30000 31.0 against 35.5 with one per CU, 16 x 4000
  // 15.7 against 18.4; head_dim 256 takes one per CU: 16 x 2000, 4 heads of 256: 15.8 against 18.4), none shorter than 256
  // tokens.
  int64_t want = 1;
  pl->W = 4;
  if (groups <= 256) {
    if (max_ctx <= 1024 || groups > 192) pl->W = 8;
    else want = std::min<int64_t>(((D == 256 ? 256 : 512) + groups - 1) / groups, ((int64_t)max_ctx + 255) / 256);
  }
  const int64_t round = pl->W * kKv4Step;                                             // tokens of a workgroup's waves at once
  const int64_t rounds = std::max<int64_t>(1, ((int64_t)max_ctx + round - 1) / round), per = (rounds + want - 1) / want;
  pl->tps = (int)(per * round);
  pl->nsplit = (int)((rounds + per - 1) / per);
  pl->ws_bytes = pl->nsplit > 1 ? (size_t)B * Hq * pl->nsplit * (D + 4) * sizeof(float) : 0;
  return 0;
}

template <class Tag, int D, int NH>
void launch_heads(const Kv4DecodeParams& p, int W, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.B * p.hgroups * p.qchunks * p.nsplit));
  if (W == 4) hipLaunchKernelGGL((kv4_decode_kernel<Tag, D, NH, 4>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((kv4_decode_kernel<Tag, D, NH, 8>), grid, dim3(512), 0, s, p);
}
template <class Tag, int D>
int launch(const Kv4DecodeParams& p, const Kv4Plan& pl, hipStream_t s) {
  switch (pl.NH) {
    case 8: if constexpr (D <= 32) launch_heads<Tag, D, 8>(p, pl.W, s); break;
    case 4: if constexpr (D <= 64) launch_heads<Tag, D, 4>(p, pl.W, s); break;
    case 2: if constexpr (D <= 128) launch_heads<Tag, D, 2>(p, pl.W, s); break;
    default: launch_heads<Tag, D, 1>(p, pl.W, s);
  }
  if (int rc = check_launch("kv4_decode_kernel")) return rc;
  if (p.nsplit > 1) {
    if (p.nsplit <= kKv4WalkedSplits) launch_merge<Tag, D, kv4_split_lanes<D>(true)>(p, s);
    else launch_merge<Tag, D, kv4_split_lanes<D>(false)>(p, s);
    return check_launch("kv4_merge_kernel");
  }
  return 0;
}
template <class Tag>
int launch(const Kv4DecodeParams& p, const Kv4Plan& pl, int D, hipStream_t s) {
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

extern "C" size_t mi355_paged_decode_kv4_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                                         int32_t max_context, int32_t dtype) {
  Kv4Plan pl;
  if (make_plan("paged_decode_kv4", B, Hq, Hkv, D, max_context, dtype, &pl)) return 0;
  return pl.ws_bytes;
}

extern "C" int mi355_paged_decode_kv4(void* out, const void* q, int64_t q_stride_seq, const void* k_cache,
                                      const void* v_cache, const int32_t* block_tables, const int32_t* context_lens,
                                      int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t block_size,
                                      int32_t max_blocks, int32_t num_blocks, int32_t max_context,
                                      int64_t stride_block, int64_t stride_head, float scale, int32_t dtype,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  if (B == 0) return 0;
  if (!out || !q || !block_tables || !context_lens) return fail(MI355_EINVAL, "paged_decode_kv4: null pointer argument");
  if (int rc = kv4_check_cache("paged_decode_kv4", k_cache, v_cache, Hkv, D, block_size, num_blocks, stride_block, stride_head))
    return rc;
  if (max_blocks <= 0) return fail(MI355_EINVAL, "paged_decode_kv4: max_blocks %d", max_blocks);
  if ((int64_t)max_context > (int64_t)max_blocks * block_size) max_context = max_blocks * block_size;
  Kv4Plan pl;
  if (int rc = make_plan("paged_decode_kv4", B, Hq, Hkv, D, max_context, dtype, &pl)) return rc;
  const int epl = dtype == MI355_F32 ? 4 : 8;
  if (q_stride_seq % epl || q_stride_seq < (int64_t)Hq * D || (((uintptr_t)q | (uintptr_t)out) & 15))
    return fail(MI355_EINVAL, "paged_decode_kv4: query rows must be 16-byte aligned and a sequence's heads packed");
  if (!kv4_out_ok(out, q, q_stride_seq, (int64_t)Hq * D, B, dtype))
    return fail(MI355_EINVAL, "paged_decode_kv4: the output overlaps the query rows without being them");
  if (pl.ws_bytes && (!workspace || workspace_bytes < pl.ws_bytes || ((uintptr_t)workspace & 15)))
    return fail(MI355_EWORKSPACE, "paged_decode_kv4: workspace of %zu bytes needed (16-byte aligned), %zu given", pl.ws_bytes,
                workspace ? workspace_bytes : (size_t)0);
  if (!kv4_grid_ok((int64_t)B * pl.hgroups * pl.qchunks * pl.nsplit, pl.W * 64) || (pl.nsplit > 1 && !kv4_grid_ok((int64_t)B * Hq, 256)) ||
      (int64_t)B * Hq > INT32_MAX)
    return fail(MI355_EINVAL, "paged_decode_kv4: too many workgroups (B=%d Hq=%d)", B, Hq);
  Kv4DecodeParams p;
  p.out = static_cast<char*>(out);
  p.q = static_cast<const char*>(q);
  p.cache = kv4_cache(k_cache, v_cache, stride_block, stride_head, num_blocks, block_size / kKv4Tile);
  p.bt = block_tables;
  p.ctx = context_lens;
  p.ws = static_cast<float*>(workspace);
  p.q_stride = q_stride_seq;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.gc = pl.gc;
  p.qchunks = pl.qchunks;
  p.hgroups = pl.hgroups;
  p.max_blocks = max_blocks;
  p.max_ctx = max_context;
  p.nsplit = pl.nsplit;
  p.tps = pl.tps;
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
