// Attention of several new query tokens per sequence over the 4-bit KV cache (their K / V rows are in
// it already): query j of a segment attends to positions 0 .. pos0 + j.
//
// The query rows of a (segment, kv head) are its (token, query head of the group) pairs; a wave owns
// MC tiles of 16 of them (the columns of its score tiles) and walks the context in steps of 32
// tokens.  A step's K and V are converted to bf16 once (exact) and serve the wave's MC tiles.
#include <algorithm>

#include "kv4.h"

namespace mi355 {
namespace {

constexpr int kWaves = 4;

struct Kv4PrefillParams {
  char* out;
  const char* q;
  Kv4Cache cache;
  const int32_t* bt;
  const int32_t* seg_q0;
  const int32_t* seg_len;
  const int32_t* seg_pos0;
  int64_t q_stride;   // elements
  int nseg, Hq, Hkv, G, max_blocks, max_ctx, row_tiles;
  float scale2;
};

template <class Tag, int D, int MC>
__global__ void __launch_bounds__(256) kv4_prefill_kernel(const Kv4PrefillParams p) {
  constexpr int NP = Kv4Pieces<Tag>::n, KS = D / 32, EB = Tag::kBytes;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  Kv4Lane<D> at(lane);
  int idx = blockIdx.x;
  const int h = idx % p.Hkv;
  idx /= p.Hkv;
  const int seg = idx % p.nseg;
  const int rt = p.row_tiles - 1 - idx / p.nseg;   // the longest contexts first
  const int len = p.seg_len[seg], pos0 = p.seg_pos0[seg], q0 = p.seg_q0[seg];
  const int rows = len * p.G;
  const int row0 = (rt * kWaves + wave) * MC * 16;
  if (row0 >= rows) return;   // (no barrier below)

  int lim[MC];       // last position the column attends to
  int64_t orow[MC];  // its row of out (and of q), -1: none
  bf16x8_t qf[MC][KS][NP];
#pragma unroll
  for (int mc = 0; mc < MC; ++mc) {
    const int r = row0 + mc * 16 + col;
    const int tok = min(r, rows - 1) / p.G, hq = h * p.G + min(r, rows - 1) % p.G;
    lim[mc] = min(pos0 + tok, p.max_ctx - 1);
    orow[mc] = r < rows ? (int64_t)(q0 + tok) * p.Hq + hq : -1;
    const char* src = p.q + ((int64_t)(q0 + tok) * p.q_stride + (int64_t)hq * D + g * (D / 4)) * EB;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
      load8<Tag>(src + s * 8 * EB, x);
      bf16_pieces<NP>(x, qf[mc][s]);
    }
  }
  const int first_lim = min(pos0 + row0 / p.G, p.max_ctx - 1);                                  // of the wave's first row
  const int last_lim = min(pos0 + min(row0 + MC * 16 - 1, rows - 1) / p.G, p.max_ctx - 1);      // of its last one

  f32x4 acc[MC][KS][2];
  float m[MC], l[MC];
#pragma unroll
  for (int mc = 0; mc < MC; ++mc) {
    m[mc] = kKv4Floor;
    l[mc] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) acc[mc][s][0] = acc[mc][s][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* table = p.bt + (int64_t)seg * p.max_blocks;
  const int last_tile = max(last_lim, 0) / kKv4Tile;
  auto record = [&](int tile) -> int64_t {
    tile = min(tile, last_tile);
    return kv4_record(p.cache, kv4_place(p.cache, table, tile), kv4_tile_bytes(D)) + (int64_t)h * p.cache.s_head;
  };

  for (int t0 = 0; t0 <= last_lim; t0 += kKv4Step) {
    Kv4TileRegs<D> T[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = record(t0 / kKv4Tile + i);
      kv4_load_k<D, false>(scalar_base(p.cache.k + r), at, T[i]);
      kv4_load_v<D, false>(scalar_base(p.cache.v + r), at, T[i]);
    }
    const bool masked = t0 + kKv4Step - 1 > first_lim;
    f32x4 S[MC][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int mc = 0; mc < MC; ++mc) S[mc][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bf16x8_t a = kv4_k_frag(T[i].k[s], kv4_k_scale<D>(T[i], at, s));
#pragma unroll
        for (int mc = 0; mc < MC; ++mc)
#pragma unroll
          for (int n = 0; n < NP; ++n) S[mc][i] = mfma_bf16(a, qf[mc][s][n], S[mc][i]);
      }
    }
    if (masked) {
      // A value row some column must not see enters with weight 0, and 0 * NaN is NaN: rows behind the
      // wave's last position count as 0, and NaN blocks are taken out of the product and added to the
      // columns that do see them.
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int first = t0 + i * kKv4Tile + 4 * g, live = last_lim + 1 - first;
        const uint32_t keep = live >= 4 ? ~0u : (live <= 0 ? 0u : (1u << (8 * live)) - 1u);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          uint32_t vs = (T[i].vs[s] & keep) | (0x7f7f7f7fu & ~keep);
          T[i].v[s] &= keep;
          uint32_t nan = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) nan |= ((vs >> (8 * j)) & 0xffu) == 255u ? 0xffu << (8 * j) : 0u;
          if (__ballot(nan != 0)) {
            vs = (vs & ~nan) | (0x7f7f7f7fu & nan);
            T[i].v[s] &= ~nan;
#pragma unroll
            for (int mc = 0; mc < MC; ++mc) {
              // (a lane's scales are those of ITS four tokens; the column needs all sixteen of the tile)
              int hit = 0;
#pragma unroll
              for (int gg = 0; gg < 4; ++gg) {
                const uint32_t other = (uint32_t)__shfl((int)nan, gg * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  hit |= ((other >> (8 * j)) & 1u) && t0 + i * kKv4Tile + 4 * gg + j <= lim[mc] ? 1 : 0;
              }
              if (hit) {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[mc][s][0][e] = acc[mc][s][1][e] = __builtin_nanf("");
              }
            }
          }
          T[i].vs[s] = vs;
        }
      }
    }
    bf16x8_t pf[MC][NP];
#pragma unroll
    for (int mc = 0; mc < MC; ++mc) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = S[mc][e >> 2][e & 3] * p.scale2;
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (t0 + (e >> 2) * kKv4Tile + 4 * g + (e & 3) > lim[mc]) x[e] = -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
      if (__ballot(top > m[mc] + kKv4Raise)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m[mc], top), f = fast_exp2(m[mc] - mn);
        m[mc] = mn;
        l[mc] *= f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          acc[mc][s][0] *= f;
          acc[mc][s][1] *= f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = fast_exp2(x[e] - m[mc]);
        l[mc] += x[e];
      }
      bf16_pieces<NP>(x, pf[mc]);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8_t ev, od;
      kv4_v_frags(T[0].v[s], T[1].v[s], T[0].vs[s], T[1].vs[s], ev, od);
#pragma unroll
      for (int mc = 0; mc < MC; ++mc)
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          acc[mc][s][0] = mfma_bf16(ev, pf[mc][n], acc[mc][s][0]);
          acc[mc][s][1] = mfma_bf16(od, pf[mc][n], acc[mc][s][1]);
        }
    }
  }

#pragma unroll
  for (int mc = 0; mc < MC; ++mc) {
    float L = l[mc];
    L += __shfl_xor(L, 16);
    L += __shfl_xor(L, 32);
    const float inv = lim[mc] >= 0 ? 1.f / L : 0.f;   // a query before position 0 sees nothing: zeros
    if (orow[mc] < 0) continue;
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

template <class Tag, int D>
int launch(const Kv4PrefillParams& p0, int max_q_len, hipStream_t s) {
  constexpr int MC = D == 256 ? 1 : 2;
  Kv4PrefillParams p = p0;
  p.row_tiles = (int)ceil_div64((int64_t)max_q_len * p.G, kWaves * MC * 16);
  const int64_t wgs = (int64_t)p.row_tiles * p.nseg * p.Hkv;
  if (wgs > INT32_MAX) return fail(MI355_EINVAL, "paged_prefill_kv4: too many workgroups");
  hipLaunchKernelGGL((kv4_prefill_kernel<Tag, D, MC>), dim3((unsigned)wgs), dim3(256), 0, s, p);
  return check_launch("kv4_prefill_kernel");
}
template <class Tag>
int launch(const Kv4PrefillParams& p, int D, int max_q_len, hipStream_t s) {
  switch (D) {
    case 32: return launch<Tag, 32>(p, max_q_len, s);
    case 64: return launch<Tag, 64>(p, max_q_len, s);
    case 128: return launch<Tag, 128>(p, max_q_len, s);
    default: return launch<Tag, 256>(p, max_q_len, s);
  }
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" size_t mi355_paged_prefill_kv4_workspace_bytes(int32_t nseg, int32_t total_rows, int32_t max_q_len,
                                                          int32_t Hq, int32_t Hkv, int32_t D, int32_t max_context,
                                                          int32_t dtype) {
  return 0;
}

extern "C" int mi355_paged_prefill_kv4(void* out, const void* q, int64_t q_stride_tok, const void* k_cache,
                                       const void* v_cache, const int32_t* block_tables, const int32_t* seg_q_start,
                                       const int32_t* seg_len, const int32_t* seg_pos0, int32_t nseg,
                                       int32_t max_q_len, int32_t Hq, int32_t Hkv, int32_t D, int32_t block_size,
                                       int32_t max_blocks, int32_t num_blocks, int32_t max_context,
                                       int64_t stride_block, int64_t stride_head, float scale, int32_t dtype,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  if (nseg == 0 || max_q_len == 0) return 0;
  if (!out || !q || !block_tables || !seg_q_start || !seg_len || !seg_pos0)
    return fail(MI355_EINVAL, "paged_prefill_kv4: null pointer argument");
  if (int rc = kv4_check_cache("paged_prefill_kv4", k_cache, v_cache, Hkv, D, block_size, num_blocks, stride_block, stride_head))
    return rc;
  if (!kv4_dtype_ok(dtype)) return fail(MI355_EINVAL, "paged_prefill_kv4: dtype %d", dtype);
  if (nseg < 0 || max_q_len < 0 || Hq <= 0 || Hq % Hkv || max_blocks <= 0 || max_context <= 0 ||
      (max_context > kKv4MaxContext && (int64_t)max_blocks * block_size > kKv4MaxContext))
    return fail(MI355_EINVAL, "paged_prefill_kv4: bad shape (nseg=%d max_q_len=%d Hq=%d Hkv=%d max_blocks=%d max_context=%d)",
                nseg, max_q_len, Hq, Hkv, max_blocks, max_context);
  if ((int64_t)max_context > (int64_t)max_blocks * block_size) max_context = max_blocks * block_size;
  if ((int64_t)max_q_len * (Hq / Hkv) > INT32_MAX) return fail(MI355_EINVAL, "paged_prefill_kv4: max_q_len %d", max_q_len);
  const int epl = dtype == MI355_F32 ? 4 : 8;
  if (q_stride_tok % epl || q_stride_tok < (int64_t)Hq * D || (((uintptr_t)q | (uintptr_t)out) & 15))
    return fail(MI355_EINVAL, "paged_prefill_kv4: query rows must be 16-byte aligned and a token's heads packed");
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
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.max_blocks = max_blocks;
  p.max_ctx = max_context;
  p.row_tiles = 0;
  p.scale2 = scale * 1.44269504088896340736f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MI355_F32: return launch<F32>(p, D, max_q_len, s);
    case MI355_BF16: return launch<BF16>(p, D, max_q_len, s);
    default: return launch<F16>(p, D, max_q_len, s);
  }
}
