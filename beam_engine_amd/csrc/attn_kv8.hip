// Paged attention over a KV cache held in 8 bits (gfx950): e4m3 codes and a
// power-of-two scale for each page, K or V, and KV head (kv8.hip).  Queries, the
// probabilities and the output are bf16 or fp16; head_dim 64, 128 or 256, any page size.
//
// One workgroup of four waves per (work item, KV head): RT 16-row tiles of the item's
// rows (queries x GQA group) over its tokens in 64-token tiles.  Codes go global -> LDS
// directly, two tiles in flight; a wave reads its MFMA operands from LDS as codes and
// turns them into 16-bit values in registers (v_cvt_scalef32_pk), so neither HBM nor
// LDS moves a 16-bit K or V.  K's scale multiplies the fp32 scores, V's the conversion:
// both exact (fp16 values of V below 2^-14 round to its subnormal step of 2^-24).
//
// Sᵀ = K Qᵀ with v_mfma_f32_16x16x32: lane (lg, lc) reads 16 codes of token lc at a
// time, which are the A operands of two products over a permuted head_dim order that Q
// follows.  The C layout of a 16-token Sᵀ tile (lane (lg, lc): tokens 4 lg .. + 3 of
// row lc) is half the B operand of Oᵀ += Vᵀ Pᵀ, two token sub-tiles to a product; Vᵀ is
// read from row-major V with ds_read_b64_tr_b8, whose eight rows are the same lanes'
// tokens of both sub-tiles.

#include <math.h>

#include <type_traits>

#include "attn_tile.h"

namespace be {
namespace kv8 {

using stream::lds_addr;
using stream::pack4;
using stream::rfl;

typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v2i* lds_v2i_t;

// Two codes of the low or high half of a word times the scale, as 16-bit values.
template <typename T, bool HIGH> __device__ __forceinline__ uint32_t value2(int codes, float scale) {
  if constexpr (std::is_same<T, bf16_t>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
}
// Eight codes without a scale.
template <typename T> __device__ __forceinline__ v8s codes8(int a, int b) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(v8s, (u4){value2<T, false>(a, 1.f), value2<T, true>(a, 1.f), value2<T, false>(b, 1.f),
                                      value2<T, true>(b, 1.f)});
}
// Two codes under a scale each.
template <typename T, bool HIGH> __device__ __forceinline__ uint32_t value11(int codes, float s0, float s1) {
  return (value2<T, HIGH>(codes, s0) & 0xffffu) | (value2<T, HIGH>(codes, s1) & 0xffff0000u);
}

// Bit 7 of every byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(int codes) {
  return (((uint32_t)codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// The value XORed into the 16-byte chunk index of row r in LDS.  Rows of CPR chunks
// fill 16 / CPR rows of all 64 banks; 16 consecutive rows' chunk (a K read's quarter
// wave) and the 16 rows 8 m .. + 7, 16 + 8 m .. + 7 (a half wave's transposed V read)
// each fall on 16 different chunk slots.
template <int CPR>
__device__ __forceinline__ int swz(int r) {
  return ((r / (16 / CPR)) & (CPR / 2 - 1)) | ((((r >> 3) ^ (r >> 4)) & 1) * (CPR / 2));
}

// Takes NaN codes out of a V tile in LDS, noting the first such token of each column:
// the rows that see it get their NaN at the end.  (By all threads of the workgroup, on
// tiles with tokens that some row must not see.)
template <int D>
__device__ __forceinline__ void set_nans_aside(unsigned char* v, int tok0, int tid, int32_t* nan_tok, int32_t* nan_any) {
  constexpr int CPR = D / 16;
#pragma unroll 1
  for (int c = tid; c < kTile * CPR; c += 256) {
    const v4i w = *reinterpret_cast<const v4i*>(v + c * 16);
    if (__builtin_expect((nan_bytes(w[0]) | nan_bytes(w[1]) | nan_bytes(w[2]) | nan_bytes(w[3])) == 0, 1)) continue;
    const int row = c / CPR, col = ((c % CPR) ^ swz<CPR>(row)) * 16;
#pragma unroll 1
    for (int b = 0; b < 16; ++b)
      if ((v[c * 16 + b] & 0x7f) == 0x7f) {
        atomicMin(&nan_tok[col + b], tok0 + row);
        v[c * 16 + b] = 0;
      }
    *nan_any = 1;
  }
}

// A row's log-sum-exp, NaN where a score was (a merge of such a part is NaN too).
__device__ __forceinline__ void store_lse(const AttnArgs& a, const WorkItem& it, int j, int head, float m2, float l) {
  const float lse = l == 0.f ? -INFINITY : (m2 + log2f(l)) * 0.69314718055994531f;
  if (it.out_row >= 0) a.part_lse[(int64_t)(it.out_row + j) * a.hq + head] = lse;
  else if (a.out_lse) a.out_lse[(int64_t)a.q_index[it.q_begin + j] * a.hq + head] = lse;
}

template <typename T, int D, int RT, bool PAGED4, bool QUADS>
__global__ __launch_bounds__(256, D == 256 ? 2 : 4) void attn_kv8_kernel(AttnArgs a) {
  constexpr int CPR = D / 16;                        // 16-code chunks of a row
  using Loader = TileLoader<D, PAGED4, swz<CPR>>;
  constexpr int PLANE = Loader::PLANE, STAGE = Loader::STAGE;
  constexpr int KP = D / 64;                         // K chunk quads: two QK contraction steps each
  constexpr int TS = RT == 4 ? 1 : 2;                // waves sharing a row tile: token halves,
  constexpr int CS = RT == 1 ? 2 : 1;                // and head_dim halves of Oᵀ
  constexpr int NSUB = 4 / TS;                       // 16-token sub-tiles per wave per tile
  constexpr int MT = D / 16 / CS;                    // Oᵀ head_dim tiles of a wave
  constexpr int COMB_SLOT = (MT * 64 * 4 + 2 * 64) * 4;
  static_assert(TS == 1 || 2 * COMB_SLOT <= 2 * STAGE, "combine scratch must fit");

  __shared__ __attribute__((aligned(1024))) unsigned char stage[2 * STAGE];
  __shared__ int32_t pg_lds[kMaxPagesLds];
  __shared__ uint16_t sc_lds[kMaxPagesLds];          // scale bytes of the pages: K | V << 8
  __shared__ int32_t nan_tok[D];                     // per column: the first masked tile's token whose V is NaN
  __shared__ int32_t nan_any;
  if (a.live_items && (int)blockIdx.x >= *a.live_items) return;

  const WorkItem it = a.items[blockIdx.x];
  const int kvh = blockIdx.y;
  const int tid = threadIdx.x;
  const int w = rfl(tid >> 6), lane = tid & 63, lg = lane >> 4, lc = lane & 15;
  const int g = a.g, R = it.q_count * g, ps = a.page_size;

  // ---- the item's pages
  const int first_page = it.tok_begin / ps;
  const int n_pages = (it.tok_begin + it.tok_count - 1) / ps - first_page + 1;
  const int n_tiles = (it.tok_count + kTile - 1) / kTile;
  const uint32_t lds0 = lds_addr(stage);
  Loader ld;
  if constexpr (PAGED4) {
    ld.init(a, it, kvh, w, pg_lds, first_page, n_pages);
    for (int i = 64 + tid; i < n_pages; i += 256) pg_lds[i] = a.pages[it.page_begin + first_page + i];
    if (tid < min(n_pages, 64)) pg_lds[tid] = ld.pg_reg;
  } else {
    for (int i = tid; i < n_pages; i += 256) pg_lds[i] = a.pages[it.page_begin + first_page + i];
    __syncthreads();
    ld.init(a, it, kvh, w, pg_lds, first_page, n_pages);
  }

  // ---- wave role
  const int rt = RT == 1 ? 0 : w % RT, ts = RT == 4 ? 0 : RT == 2 ? w >> 1 : w & 1, cs = RT == 1 ? w >> 1 : 0;
  const bool active = rt * 16 < R;
  const int row = rt * 16 + lc;
  // row / g for row < 256 (the quotient's distance from an integer is at least 1 / (2 g))
  const int j = (int)(((float)row + 0.5f) * (1.f / (float)g)), hh = row - j * g;

  // ---- Q as the B operand: product 2 kp + i takes head_dim 16 (4 kp + lg) + 8 i .. + 7
  v8s qf[2 * KP];
  if (row < R) {
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(it.q_begin + j) * a.q_sn + (int64_t)(kvh * g + hh) * a.q_sh;
#pragma unroll
    for (int x = 0; x < 2 * KP; ++x) qf[x] = *reinterpret_cast<const v8s*>(qp + 16 * (4 * (x >> 1) + lg) + 8 * (x & 1));
  } else {
#pragma unroll
    for (int x = 0; x < 2 * KP; ++x) qf[x] = v8s{0, 0, 0, 0, 0, 0, 0, 0};
  }
#pragma unroll
  for (int x = 0; x < 2 * KP; ++x) asm volatile("" : "+v"(qf[x]));
  ld.load(lds0);
  if (n_tiles > 1) ld.load(lds0 + STAGE);
  for (int i = tid; i < D; i += 256) nan_tok[i] = INT32_MAX;
  if (tid == 0) nan_any = 0;
  // ---- the pages' scales (behind the first tiles' loads, which they need not precede)
  for (int i = tid; i < n_pages; i += 256) {
    const int64_t at = (int64_t)a.pages[it.page_begin + first_page + i] * 2 * a.hkv + kvh;
    sc_lds[i] = (uint16_t)(a.kv_scale[at] | (uint32_t)a.kv_scale[at + a.hkv] << 8);
  }
  // page of the item's token t: pages hold at most 1024 tokens and an item 1024 pages
  const int slot0 = it.tok_begin - first_page * ps;
  const float inv_ps = 1.f / (float)ps;
  auto page_of = [&](int t) { return min((int)(((float)(slot0 + t) + 0.5f) * inv_ps), n_pages - 1); };
  auto k_scale = [&](int t) { return __uint_as_float((uint32_t)(sc_lds[page_of(t)] & 0xff) << 23); };
  auto v_scale = [&](int t) { return __uint_as_float((uint32_t)(sc_lds[page_of(t)] >> 8) << 23); };
  // item tokens this lane's row sees (causal: its query's limit)
  int lim;
  {
    const int64_t v = (int64_t)it.vis0 + j - it.tok_begin;
    lim = (int)std::min<int64_t>(it.tok_count, std::max<int64_t>(v, 0));
  }
  // ---- operand offsets of sub-tile pairs (the swizzle repeats every 32 rows)
  uint32_t koff[2][KP], voff[MT];
#pragma unroll
  for (int o = 0; o < 2; ++o)
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) koff[o][kp] = (16 * o + lc) * D + (((4 * kp + lg) ^ swz<CPR>(16 * o + lc)) << 4);
  const int vj = lc >> 1, vr = (vj >> 2) * 16 + 4 * lg + (vj & 3);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) voff[mt] = vr * D + (((cs * MT + mt) ^ swz<CPR>(vr)) << 4) + (lc & 1) * 8;

  // item tokens from here on are not seen by the first query (causal)
  const int unseen = (int)std::min<int64_t>(it.tok_count, std::max<int64_t>((int64_t)it.vis0 - it.tok_begin, 0));
  float m_run = -INFINITY, l_run = 0.f;
  v4f o_acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) o_acc[mt] = v4f{0.f, 0.f, 0.f, 0.f};

  for (int tile = 0; tile < n_tiles; ++tile) {
    const int st = tile & 1;
    // this wave's loads of the tile have landed (the next tile's may be in
    // flight); after the barrier everyone's have
    if (tile + 1 < n_tiles) {
      if constexpr (Loader::IPW == 1) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else if constexpr (Loader::IPW == 2) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if (unseen < min(it.tok_count, (tile + 1) * kTile)) {
      // tokens that a row must not see: their NaN would reach it by a weight of 0
      set_nans_aside<D>(stage + st * STAGE + PLANE, tile * kTile, tid, nan_tok, &nan_any);
      stream::lds_sync();
    }
    const int s0 = tile * kTile + ts * NSUB * 16;      // first token of the wave's sub-tiles
    if (active && s0 < it.tok_count) {
      const unsigned char* kt = stage + st * STAGE + ts * NSUB * 16 * D;
      const unsigned char* vt = kt + PLANE;
      float x[NSUB][4];
#pragma unroll
      for (int k = 0; k < NSUB; ++k) {
        v4i kc[KP];
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) kc[kp] = *reinterpret_cast<const v4i*>(kt + (k >> 1) * 32 * D + koff[k & 1][kp]);
        float ks[QUADS ? 1 : 4];                       // of the lane's four tokens in the C layout
#pragma unroll
        for (int r = 0; r < (QUADS ? 1 : 4); ++r) ks[r] = k_scale(s0 + k * 16 + 4 * lg + r) * a.scale_log2;
        v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
          acc = mfma_qk<T>(codes8<T>(kc[kp][0], kc[kp][1]), qf[2 * kp], acc);
          acc = mfma_qk<T>(codes8<T>(kc[kp][2], kc[kp][3]), qf[2 * kp + 1], acc);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) x[k][r] = acc[r] * ks[QUADS ? 0 : r];
      }
      if (__builtin_amdgcn_ballot_w64(lim < s0 + NSUB * 16) != 0) {
        const int left = lim - s0 - 4 * lg;
#pragma unroll
        for (int k = 0; k < NSUB; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (k * 16 + r >= left) x[k][r] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < NSUB; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[k][r]);
      mx = rows4_max(mx);
      const float m_new = fmaxf(m_run, mx);
      const float msafe = (m_new == -INFINITY) ? 0.f : m_new;
      if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0) {
        const float alpha = __builtin_amdgcn_exp2f(m_run - msafe);    // 0 while nothing was seen
        l_run *= alpha;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o_acc[mt] *= alpha;
      }
      m_run = m_new;
      v4s pf[NSUB];
#pragma unroll
      for (int k = 0; k < NSUB; ++k) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = __builtin_amdgcn_exp2f(x[k][r] - msafe);
          l_run += p[r];
        }
        pf[k] = pack4<T>(p[0], p[1], p[2], p[3]);
      }
#pragma unroll
      for (int k = 0; k < NSUB; k += 2) {
        const v8s pb = __builtin_shufflevector(pf[k], pf[k + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        // scales of the lane's eight tokens: 4 lg .. + 3 of both sub-tiles
        float vs[2][QUADS ? 1 : 4];
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
          for (int r = 0; r < (QUADS ? 1 : 4); ++r) vs[o][r] = v_scale(s0 + (k + o) * 16 + 4 * lg + r);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const v2i vc = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i_t)(vt + k * 16 * D + voff[mt]));
          typedef uint32_t u4 __attribute__((ext_vector_type(4)));
          u4 vv;
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            if constexpr (QUADS) {
              vv[2 * o] = value2<T, false>(vc[o], vs[o][0]);
              vv[2 * o + 1] = value2<T, true>(vc[o], vs[o][0]);
            } else {
              vv[2 * o] = value11<T, false>(vc[o], vs[o][0], vs[o][1]);
              vv[2 * o + 1] = value11<T, true>(vc[o], vs[o][2], vs[o][3]);
            }
          }
          o_acc[mt] = mfma_qk<T>(__builtin_bit_cast(v8s, vv), pb, o_acc[mt]);
        }
      }
    }
    if (tile + 2 < n_tiles) {
      // everyone is done with this stage
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      ld.load(lds0 + st * STAGE);
    }
  }
  l_run = rows4_sum(l_run);

  // ---- the second token half hands its state to the first
  if constexpr (TS > 1) {
    float* comb = reinterpret_cast<float*>(stage);
    const int pair = RT == 2 ? rt : cs;
    __syncthreads();                                   // tiles no longer needed
    if (ts > 0 && active) {
      float* slot = comb + pair * (COMB_SLOT / 4);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<v4f*>(slot + (mt * 64 + lane) * 4) = o_acc[mt];
      slot[MT * 256 + lane] = m_run;
      slot[MT * 256 + 64 + lane] = l_run;
    }
    __syncthreads();
    if (ts == 0 && active) {
      const float* slot = comb + pair * (COMB_SLOT / 4);
      const float mb = slot[MT * 256 + lane], lb = slot[MT * 256 + 64 + lane];
      const float M = fmaxf(m_run, mb);
      const float ca = (M == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(m_run - M);
      const float cb = (M == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(mb - M);
      l_run = l_run * ca + lb * cb;
      m_run = M;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        o_acc[mt] = o_acc[mt] * ca + *reinterpret_cast<const v4f*>(slot + (mt * 64 + lane) * 4) * cb;
    }
  }

  // ---- writes: lane holds Oᵀ[16 (cs MT + mt) + 4 lg + i][row]
  if (ts == 0 && active && row < R) {
    const int head = kvh * g + hh, d0 = cs * MT * 16;
    const float inv = (l_run > 0.f) ? 1.f / l_run : 0.f;
    if (nan_any) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (nan_tok[d0 + mt * 16 + 4 * lg + r] < lim) o_acc[mt][r] = NAN;
    }
    if (it.out_row < 0) {
      T* op = reinterpret_cast<T*>(a.out) + (int64_t)(it.q_begin + j) * a.o_sn + (int64_t)head * a.o_sh + d0;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        *reinterpret_cast<v4s*>(op + mt * 16 + 4 * lg) =
            pack4<T>(o_acc[mt][0] * inv, o_acc[mt][1] * inv, o_acc[mt][2] * inv, o_acc[mt][3] * inv);
    } else {
      float* op = a.part_o + ((int64_t)(it.out_row + j) * a.hq + head) * D + d0;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<v4f*>(op + mt * 16 + 4 * lg) = o_acc[mt] * inv;
    }
    if (lg == 0 && cs == 0) store_lse(a, it, j, head, m_run, l_run);
  }
}

template <typename T, int D, int RT>
static void launch_rt(const AttnArgs& a, dim3 grid, hipStream_t st) {
  if (paged4(a.page_size, D) && a.page_size % 4 == 0) attn_kv8_kernel<T, D, RT, true, true><<<grid, 256, 0, st>>>(a);
  else if (a.page_size % 4 == 0) attn_kv8_kernel<T, D, RT, false, true><<<grid, 256, 0, st>>>(a);
  else attn_kv8_kernel<T, D, RT, false, false><<<grid, 256, 0, st>>>(a);
}

template <typename T, int D>
static int launch_tile(const be_attn_plan_info* info, const AttnArgs& a, hipStream_t st) {
  const dim3 grid(info->grid_items, info->num_kv_heads);
  switch (info->tile_rows) {
    case 16: launch_rt<T, D, 1>(a, grid, st); break;
    case 32: launch_rt<T, D, 2>(a, grid, st); break;
    case 64: launch_rt<T, D, 4>(a, grid, st); break;
    default: return fail(BE_ERR_INVALID, "corrupt plan: tile_rows %d", info->tile_rows);
  }
  BE_HIP_CHECK(hipGetLastError());
  return BE_OK;
}

template <typename T>
static int launch_d(const be_attn_plan_info* info, const AttnArgs& a, hipStream_t st) {
  switch (info->head_dim) {
    case 64: return launch_tile<T, 64>(info, a, st);
    case 128: return launch_tile<T, 128>(info, a, st);
    case 256: return launch_tile<T, 256>(info, a, st);
    default: return fail(BE_ERR_UNSUPPORTED, "head_dim %d", info->head_dim);
  }
}

}  // namespace kv8

int kv8_launch(const be_attn_plan_info* info, const AttnArgs& a, hipStream_t st) {
  return info->dtype == BE_BF16 ? kv8::launch_d<bf16_t>(info, a, st) : kv8::launch_d<f16_t>(info, a, st);
}

}  // namespace be
