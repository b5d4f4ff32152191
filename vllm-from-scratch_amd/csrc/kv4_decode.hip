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
// The four waves of a workgroup take steps in turn and combine their sums in LDS; a long context is
// split over workgroups, whose partial sums kv4_merge_kernel joins.
#include <algorithm>

#include "kv4.h"

namespace mi355 {
namespace {

constexpr int kWaves = 4;

struct Kv4DecodeParams {
  char* out;
  const char* q;
  Kv4Cache cache;
  const int32_t* bt;
  const int32_t* ctx;
  float* ws_acc;   // [B * Hq][nsplit][D]
  float* ws_ml;    // [B * Hq][nsplit][2]
  int64_t q_stride;   // elements
  int B, Hq, Hkv, G /* query heads per kv head */, gc /* of them per workgroup */, qchunks, hgroups;
  int max_blocks, max_ctx, nsplit, tps /* tokens per split */;
  float scale2;   // scale * log2(e)
};

template <class Tag, int D, int NH>
__global__ void __launch_bounds__(256) kv4_decode_kernel(const Kv4DecodeParams p) {
  constexpr int NP = Kv4Pieces<Tag>::n, KS = D / 32, EB = Tag::kBytes;
  __shared__ float s_o[kWaves][16][D + 4];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  int idx = blockIdx.x;
  const int sp = idx % p.nsplit;
  idx /= p.nsplit;
  const int qc = idx % p.qchunks;
  idx /= p.qchunks;
  const int hg = idx % p.hgroups, b = idx / p.hgroups;
  const int h0 = hg * NH, nh = min(NH, p.Hkv - h0);
  // column -> (kv head h0 + my_j, query head of its group)
  const int my_j = col / p.gc, my_q = qc * p.gc + col % p.gc;
  const bool used = my_j < nh && my_q < p.G;
  const int hq = (h0 + my_j) * p.G + my_q;

  int ctx = min(p.ctx[b], p.max_ctx);
  const int lo = sp * p.tps, hi = min(ctx, lo + p.tps);   // this workgroup's tokens
  if (lo >= hi && !(sp == 0 && p.nsplit == 1)) return;    // (the merge knows which splits are empty)

  bf16x8_t qf[KS][NP];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (used) load8<Tag>(p.q + ((int64_t)b * p.q_stride + (int64_t)hq * D + g * (D / 4) + s * 8) * EB, x);
    bf16_pieces<NP>(x, qf[s]);
  }
  f32x4 acc[NH][KS][2];
#pragma unroll
  for (int j = 0; j < NH; ++j)
#pragma unroll
    for (int s = 0; s < KS; ++s) acc[j][s][0] = acc[j][s][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kKv4Floor, l = 0.f;

  const int32_t* table = p.bt + (int64_t)b * p.max_blocks;
  const int last_tile = hi > 0 ? (hi - 1) / kKv4Tile : 0;
  auto record = [&](int tile) -> int64_t {   // byte offset of a tile's record of kv head h0
    tile = min(tile, last_tile);             // (a step's second tile may lie beyond the context: read the last one)
    int id = table[tile / p.cache.tpb];
    id = id < 0 ? 0 : (id >= p.cache.num_blocks ? p.cache.num_blocks - 1 : id);
    return (int64_t)id * p.cache.s_blk + (int64_t)h0 * p.cache.s_head + (tile % p.cache.tpb) * kv4_tile_bytes(D);
  };

  for (int t0 = lo + wave * kKv4Step; t0 < hi; t0 += kWaves * kKv4Step) {
    const int64_t r0 = record(t0 / kKv4Tile), r1 = record(t0 / kKv4Tile + 1);
    f32x4 S[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    Kv4TileRegs<D> T[NH][2];
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      if (j < nh) {
        kv4_load_k<D>(p.cache.k + r0 + j * p.cache.s_head, lane, T[j][0]);
        kv4_load_k<D>(p.cache.k + r1 + j * p.cache.s_head, lane, T[j][1]);
      }
    }
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      if (j < nh) {
        kv4_load_v<D>(p.cache.v + r0 + j * p.cache.s_head, lane, T[j][0]);
        kv4_load_v<D>(p.cache.v + r1 + j * p.cache.s_head, lane, T[j][1]);
      }
    }
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      if (j < nh) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x4 c = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const bf16x8_t a = kv4_k_frag(T[j][i].k[s], kv4_scale(T[j][i].ks, D == 256 ? s / 4 : 0));
#pragma unroll
            for (int n = 0; n < NP; ++n) c = mfma_bf16(a, qf[s][n], c);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) S[i][e] = my_j == j ? c[e] : S[i][e];
        }
      }
    }
    // tokens 4 g + e of each tile, in powers of two
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = S[e >> 2][e & 3] * p.scale2;
    if (t0 + kKv4Step > hi) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (t0 + (e >> 2) * kKv4Tile + 4 * g + (e & 3) >= hi) x[e] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < NH; ++j) {
        if (j < nh) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // rows behind the context hold whatever was there: their codes count as 0 and their scales as 1
            const int live = hi - (t0 + i * kKv4Tile + 4 * g);   // tokens of this lane's four that count
            const uint32_t keep = live >= 4 ? ~0u : (live <= 0 ? 0u : (1u << (8 * live)) - 1u);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              T[j][i].v[s] &= keep;
              T[j][i].vs[s] = (T[j][i].vs[s] & keep) | (0x7f7f7f7fu & ~keep);
            }
          }
        }
      }
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
    if (__ballot(top > m + kKv4Raise)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top), f = fast_exp2(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int j = 0; j < NH; ++j)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          acc[j][s][0] *= f;
          acc[j][s][1] *= f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = fast_exp2(x[e] - m);
      l += x[e];
    }
    bf16x8_t pf[NP];
    bf16_pieces<NP>(x, pf);
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      if (j < nh) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bf16x8_t ev, od;
          kv4_v_frags(T[j][0].v[s], T[j][1].v[s], T[j][0].vs[s], T[j][1].vs[s], ev, od);
#pragma unroll
          for (int n = 0; n < NP; ++n) {
            acc[j][s][0] = mfma_bf16(ev, pf[n], acc[j][s][0]);
            acc[j][s][1] = mfma_bf16(od, pf[n], acc[j][s][1]);
          }
        }
      }
    }
  }

  // the lane's column: dims 32 s + 8 g .. + 8 (even and odd rows of the two accumulators alternate)
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) {
    s_m[wave][col] = m;
    s_l[wave][col] = l;
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
  for (int item = threadIdx.x; item < 16 * P; item += 256) {
    const int c = item / P, d = (item % P) * 8;
    const int j = c / p.gc, qi = qc * p.gc + c % p.gc;
    if (j >= nh || qi >= p.G) continue;
    float M = s_m[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w][c]);
    float L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = fast_exp2(s_m[w][c] - M);
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
      float* dst = p.ws_acc + (row * p.nsplit + sp) * D + d;
      *reinterpret_cast<f32x4*>(dst) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(dst + 4) = f32x4{o[4], o[5], o[6], o[7]};
      if (d == 0) {
        p.ws_ml[(row * p.nsplit + sp) * 2] = M;
        p.ws_ml[(row * p.nsplit + sp) * 2 + 1] = L;
      }
    }
  }
}

// Joins the splits of a row: thread = eight dims.
template <class Tag, int D>
__global__ void __launch_bounds__(256)
kv4_merge_kernel(char* out, const float* ws_acc, const float* ws_ml, const int32_t* ctx_lens, int rows, int Hq,
                 int max_ctx, int nsplit, int tps) {
  constexpr int P = D / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / P;
  const int d = (int)(idx % P) * 8;
  if (row >= rows) return;
  const int ctx = min(ctx_lens[row / Hq], max_ctx);
  const int n = ctx <= 0 ? 0 : min(nsplit, (ctx + tps - 1) / tps);
  float M = kKv4Floor, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n; ++s) {
    const float ms = ws_ml[(row * nsplit + s) * 2], ls = ws_ml[(row * nsplit + s) * 2 + 1];
    const float* a = ws_acc + (row * nsplit + s) * D + d;
    const f32x4 lo = *reinterpret_cast<const f32x4*>(a), hi = *reinterpret_cast<const f32x4*>(a + 4);
    const float Mn = fmaxf(M, ms), fo = fast_exp2(M - Mn), fn = fast_exp2(ms - Mn);
    M = Mn;
    L = __builtin_fmaf(ls, fn, L * fo);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = __builtin_fmaf(lo[e], fn, o[e] * fo);
      o[4 + e] = __builtin_fmaf(hi[e], fn, o[4 + e] * fo);
    }
  }
  const float inv = n > 0 ? 1.f / L : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] *= inv;
  store8<Tag>(out + (row * D + d) * Tag::kBytes, o);
}

struct Kv4Plan {
  int NH, gc, qchunks, hgroups, nsplit, tps;
  size_t ws_bytes;
};

// Host arithmetic only.
int make_plan(const char* what, int B, int Hq, int Hkv, int D, int max_ctx, int dtype, Kv4Plan* pl) {
  if (!kv4_dtype_ok(dtype)) return fail(MI355_EINVAL, "%s: dtype %d", what, dtype);
  if (!kv4_head_dim_ok(D)) return fail(MI355_EUNSUPPORTED, "%s: head_dim %d (the 4-bit cache holds 32, 64, 128 or 256)", what, D);
  if (B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || max_ctx < 0)
    return fail(MI355_EINVAL, "%s: bad shape (B=%d Hq=%d Hkv=%d max_context=%d)", what, B, Hq, Hkv, max_ctx);
  const int G = Hq / Hkv;
  pl->gc = std::min(G, 16);
  pl->qchunks = (G + 15) / 16;
  pl->NH = 1;
  pl->hgroups = (Hkv + pl->NH - 1) / pl->NH;
  const int64_t groups = (int64_t)std::max(B, 1) * pl->hgroups * pl->qchunks;
  const int steps = std::max(1, (max_ctx + kWaves * kKv4Step - 1) / (kWaves * kKv4Step));   // rounds of a workgroup's four waves
  int64_t want = std::max<int64_t>(1, (1024 + groups - 1) / groups);
  want = std::min<int64_t>(want, steps);
  const int per = (int)((steps + want - 1) / want);
  pl->tps = per * kWaves * kKv4Step;
  pl->nsplit = (steps + per - 1) / per;
  pl->ws_bytes = pl->nsplit > 1 ? (size_t)B * Hq * pl->nsplit * (D + 2) * sizeof(float) : 0;
  return 0;
}

template <class Tag, int D>
int launch(const Kv4DecodeParams& p, const Kv4Plan& pl, hipStream_t s) {
  const int64_t wgs = (int64_t)p.B * p.hgroups * p.qchunks * p.nsplit;
  const dim3 grid((unsigned)wgs), block(256);
  hipLaunchKernelGGL((kv4_decode_kernel<Tag, D, 1>), grid, block, 0, s, p);
  if (int rc = check_launch("kv4_decode_kernel")) return rc;
  if (p.nsplit > 1) {
    const int rows = p.B * p.Hq;
    hipLaunchKernelGGL((kv4_merge_kernel<Tag, D>), dim3((unsigned)ceil_div64((int64_t)rows * (D / 8), 256)), block, 0, s,
                       p.out, p.ws_acc, p.ws_ml, p.ctx, rows, p.Hq, p.max_ctx, p.nsplit, p.tps);
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
  if (pl.ws_bytes && (!workspace || workspace_bytes < pl.ws_bytes || ((uintptr_t)workspace & 15)))
    return fail(MI355_EWORKSPACE, "paged_decode_kv4: workspace of %zu bytes needed (16-byte aligned), %zu given", pl.ws_bytes,
                workspace ? workspace_bytes : (size_t)0);
  if ((int64_t)B * pl.hgroups * pl.qchunks * pl.nsplit > INT32_MAX || (int64_t)B * Hq > INT32_MAX)
    return fail(MI355_EINVAL, "paged_decode_kv4: too many workgroups (B=%d Hq=%d)", B, Hq);
  Kv4DecodeParams p;
  p.out = static_cast<char*>(out);
  p.q = static_cast<const char*>(q);
  p.cache = Kv4Cache{static_cast<char*>(const_cast<void*>(k_cache)), static_cast<char*>(const_cast<void*>(v_cache)),
                     stride_block, stride_head, num_blocks, block_size / kKv4Tile};
  p.bt = block_tables;
  p.ctx = context_lens;
  p.ws_acc = static_cast<float*>(workspace);
  p.ws_ml = p.ws_acc ? p.ws_acc + (size_t)B * Hq * pl.nsplit * D : nullptr;
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
  p.scale2 = scale * 1.44269504088896340736f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MI355_F32: return launch<F32>(p, pl, D, s);
    case MI355_BF16: return launch<BF16>(p, pl, D, s);
    default: return launch<F16>(p, pl, D, s);
  }
}
