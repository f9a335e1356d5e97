// Paged attention over a KV cache held in 8 bits (gfx950): e4m3 codes and a
// power-of-two scale for each page, K or V, and KV head (kv8.hip).  Queries, the
// probabilities and the output are bf16 or fp16; head_dim 64, 128 or 256, any page size.
//
// One workgroup of four waves per (work item, KV head): RT 16-row tiles of the item's
// rows (queries x GQA group) over its tokens in 64-token tiles.  Codes go global -> LDS
// directly, two tiles ahead; a wave reads its MFMA operands from LDS as codes and
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
//
// Scores, the softmax's maxima and sums, the outputs' sums and split partials are fp32.
// Rounded once each, as the matrix instructions take them: a weight P to 16 bits (half a
// step, up to 2^-8 of it in bf16, 2^-11 in fp16; its sum is taken before), which is what the
// error against 64 bits consists of (2.3e-3 and 2.5e-4 in the 2-norm, of which the
// output's own rounding is 1.7e-3 and 2.1e-4).
//
// The products stay 16-bit: the matrix instructions that take e4m3 operands sum up to
// 2^-12.7 of the absolute sum off (measured over 64 products, against 64 bits), where
// these sums are to be good to fp32, and would need P in 8 bits.  So a code costs a
// conversion (5 cycles a wave instruction for two codes of 64 lanes), which bounds the
// tiles: 2.0 to 2.4 thousand cycles for 64 tokens x 64 rows at head_dim 128 alone on a
// CU, of which the loads' latency is a third.  Measured, with the merge: 16 sequences of
// up to 6000 tokens (32 heads of 128 over 8) 30 us, 3.2 TB/s of codes where a copy moves
// 4.9; 8 x 16 beams on 4096 shared tokens + 128 own ones 36 us, 2.9 TB/s; 2 x 64 beams
// on 32768 + 512 (64 heads over 8) 185 us, 750 TFLOP/s of the 1170 of a large 16-bit
// matrix product; 8 x 16 beams on 1136 + up to 24 20 us, where launches, a workgroup's
// start (its record, pages, scales and first tile are round trips in a row, 3 us) and the
// merge (4.4 us) are most of it.

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
// Eight codes times the scale.
template <typename T> __device__ __forceinline__ v8s codes8(int a, int b, float scale = 1.f) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(v8s, (u4){value2<T, false>(a, scale), value2<T, true>(a, scale), value2<T, false>(b, scale),
                                      value2<T, true>(b, scale)});
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
template <int D, int (*SWZ)(int)>
__device__ __forceinline__ void set_nans_aside(unsigned char* v, int tok0, int tid, int32_t* nan_tok, int32_t* nan_any) {
  constexpr int CPR = D / 16;
#pragma unroll 1
  for (int c = tid; c < kTile * CPR; c += 256) {
    const v4i w = *reinterpret_cast<const v4i*>(v + c * 16);
    if (__builtin_expect((nan_bytes(w[0]) | nan_bytes(w[1]) | nan_bytes(w[2]) | nan_bytes(w[3])) == 0, 1)) continue;
    const int row = c / CPR, col = ((c % CPR) ^ SWZ(row)) * 16;
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

// What a workgroup keeps in LDS.
template <int D> struct TileShared {
  static constexpr int kStages = D == 256 ? 2 : 3;   // tiles in LDS
  unsigned char stage[kStages * 2 * kTile * D];
  int32_t pg[kMaxPagesKv8];
  uint32_t ks[kMaxPagesKv8], vs[kMaxPagesKv8];       // scale bytes of the pages
  int32_t nan_tok[D];                  // per column: the first masked tile's token whose V is NaN
  int32_t nan_any;
};
static_assert(kMaxPagesKv8 == 256, "a thread stages one page");

// One byte a lane, global -> LDS dwords lds + 4 lane (zero-extended), as stream::dma16.
__device__ __forceinline__ void dma_byte(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
}

// 16 bytes a lane from a wave-uniform base and a byte offset, as stream::dma16_sv.
__device__ __forceinline__ void dma16_s(uint64_t base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

// An item's pages: ids and scale bytes to LDS, and the K and V codes of its tiles,
// global -> LDS directly.  The chain of a workgroup's start is three round trips: the
// item's record, page ids (with Q), scales and the first tiles.  The scales leave ahead
// of the tiles, so a wait for the first tile is one for them.
//
// PG 2: page sizes that are multiples of 16, the rows a wave loads of a tile: one page,
// whose id comes from a register (64 of the item's ids) by v_readlane, and a scalar
// address.  PG 1: multiples of a load's rows (1 KB), each load's page so.  PG 0: every
// lane looks its row's page up in LDS.  Past the item's end K re-reads its last token
// (the scores are masked) and V reads zeros.
template <int D, int PG, int (*SWZ)(int)>
struct Codes {
  static constexpr bool PAGED = PG > 0;
  static constexpr int CPR = D / 16, RPI = 64 / CPR;   // 16-byte chunks per row, rows per wave load
  static constexpr int IPW = kTile / RPI / 4;          // loads per wave per tile (K and V each)
  static constexpr int PLANE = kTile * D, STAGE = 2 * PLANE;

  uint64_t kvb;
  uint32_t row_bytes, page_bytes, vplane, off[IPW];
  int tid, w, lane, ps, tok_count, slot0, n_pages, tok;
  float inv_ps;
  int page[IPW], slot[IPW], dpage, dslot;              // PAGED: of the next tile's loads
  int id, pg_reg, pg_base;
  const int32_t* pg_lds;

  // Page of the item's token t: pages hold at most 1024 tokens and an item 256 pages.
  __device__ __forceinline__ int page_of(int t) const {
    return min((int)(((float)(slot0 + t) + 0.5f) * inv_ps), n_pages - 1);
  }

  // The page ids leave; nothing waits for them yet.
  __device__ __forceinline__ void begin(const AttnArgs& a, const WorkItem& it, int kvh, int thread) {
    tid = thread;
    w = rfl(tid >> 6);
    lane = tid & 63;
    ps = a.page_size;
    inv_ps = 1.f / (float)ps;
    tok_count = it.tok_count;
    slot0 = it.tok_begin - it.first_page * ps;
    n_pages = (int)(((float)(slot0 + tok_count - 1) + 0.5f) * inv_ps) + 1;
    const int32_t* pages = a.pages + it.page_begin + it.first_page;
    id = pages[min(tid, n_pages - 1)];
    pg_reg = PAGED ? pages[min(lane, n_pages - 1)] : 0;
    row_bytes = (uint32_t)a.hkv * D;
    vplane = (uint32_t)ps * row_bytes;
    page_bytes = 2 * vplane;
    kvb = reinterpret_cast<uint64_t>(a.kv) + (uint64_t)kvh * D;
    tok = 0;
    pg_base = 0;
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int lr = lane / CPR;
      off[i] = (uint32_t)((PG == 2 ? i * RPI : 0) + lr) * row_bytes + ((uint32_t)((lane % CPR) ^ SWZ((w * IPW + i) * RPI + lr)) << 4);
    }
    if constexpr (PAGED) {
      dpage = rfl((int)(((float)kTile + 0.5f) * inv_ps));
      dslot = kTile - dpage * ps;
#pragma unroll
      for (int i = 0; i < (PG == 2 ? 1 : IPW); ++i) {
        const int t = slot0 + (w * IPW + i) * RPI;
        page[i] = rfl((int)(((float)t + 0.5f) * inv_ps));
        slot[i] = t - page[i] * ps;
      }
    }
  }

  // Ids to LDS, scales on their way there.
  __device__ __forceinline__ void stage(const AttnArgs& a, int kvh, int32_t* pg, uint32_t* ks, uint32_t* vs) {
    pg[tid] = id;
    pg_lds = pg;
    const uint8_t* sc = a.kv_scale + (int64_t)id * 2 * a.hkv + kvh;
    dma_byte(sc, lds_addr(ks) + w * 256);
    dma_byte(sc + a.hkv, lds_addr(vs) + w * 256);
    if constexpr (!PAGED) __syncthreads();
  }

  // Scalar address of a row of the wave's pages.
  __device__ __forceinline__ uint64_t base_of(int pg, int sl) const {
    const uint32_t pid = (uint32_t)__builtin_amdgcn_readlane(pg_reg, pg - pg_base);
    return kvb + (uint64_t)pid * page_bytes + (uint32_t)sl * row_bytes;
  }
  __device__ __forceinline__ void advance(int i) {
    slot[i] += dslot;
    const bool carry = slot[i] >= ps;
    slot[i] -= carry ? ps : 0;
    page[i] += dpage + (carry ? 1 : 0);
  }

  __device__ __forceinline__ void whole(uint32_t dst0) {
    dst0 += w * IPW * 1024;
    if constexpr (PG == 2) {
      const uint64_t base = base_of(page[0], slot[0]);
#pragma unroll
      for (int i = 0; i < IPW; ++i) dma16_s(base, off[i], dst0 + i * 1024);
#pragma unroll
      for (int i = 0; i < IPW; ++i) dma16_s(base + vplane, off[i], dst0 + i * 1024 + PLANE);
      advance(0);
    } else if constexpr (PG == 1) {
#pragma unroll
      for (int i = 0; i < IPW; ++i) {
        const uint64_t base = base_of(page[i], slot[i]);
        dma16_s(base, off[i], dst0 + i * 1024);
        dma16_s(base + vplane, off[i], dst0 + i * 1024 + PLANE);
        advance(i);
      }
    } else {
      any(dst0);
    }
  }
  // Any tile, row by row.
  __device__ __forceinline__ void any(uint32_t dst) {
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int r = (w * IPW + i) * RPI + lane / CPR;
      const bool in = tok + r < tok_count;
      const int t = in ? tok + r : tok_count - 1, pg = page_of(t), sl = slot0 + t - pg * ps;
      const uint32_t pid = PAGED ? (uint32_t)__shfl(pg_reg, pg - pg_base) : (uint32_t)pg_lds[pg];
      const uint64_t src = kvb + (uint64_t)pid * page_bytes + (uint32_t)sl * row_bytes + ((uint32_t)((lane % CPR) ^ SWZ(r)) << 4);
      stream::dma16(reinterpret_cast<const void*>(src), dst + i * 1024);
      stream::dma16(in ? reinterpret_cast<const void*>(src + vplane) : &kZeroChunk, dst + i * 1024 + PLANE);
    }
  }

  // The next tile's loads, to LDS byte address dst0 (2 IPW vector memory operations).
  __device__ __forceinline__ void load(uint32_t dst0) {
    if constexpr (PAGED) {
      // (the wave's pages of a tile lie within 64 of its first; pg_lds is read from the third
      // tile on, behind a barrier: the first two lie within the register's first 64 pages)
      const int last = n_pages - 1, p1 = min(page[PG == 2 ? 0 : IPW - 1], last);
      if (p1 - pg_base >= 64) {
        pg_base = min(page[0], last);
        pg_reg = pg_lds[min(pg_base + lane, last)];
      }
    }
    if (__builtin_expect(tok + kTile <= tok_count, 1)) whole(dst0);
    else any(dst0 + w * IPW * 1024);
    tok += kTile;
  }

  // Waits until the tile that was loaded `newer` loads ago is whole, for everyone.
  template <int newer> static __device__ __forceinline__ void wait() {
    constexpr int N = 2 * IPW * newer;
    if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
};

// Consecutive workgroups are the KV heads of one item: an XCD keeps the same heads in its
// L2, and the items start in their order.  x / hkv by the reciprocal, which is at most
// one too large (a division by a variable costs a start some 200 cycles).
__device__ __forceinline__ int item_of(const AttnArgs& a, uint32_t x) {
  if (a.hkv == 1) return (int)x;
  const uint32_t i = __umulhi(x, a.hkv_inv);
  return (int)(i * (uint32_t)a.hkv > x ? i - 1 : i);
}

// An item's record by scalar loads, whatever the compiler can tell of its index.
__device__ __forceinline__ WorkItem item_at(const AttnArgs& a, int i) {
  typedef const int32_t __attribute__((address_space(4)))* words_t;
  const words_t p = (words_t)reinterpret_cast<uint64_t>(a.items + rfl(i));
  return WorkItem{p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]};
}

// The item in each of a kernel's branches by itself: what they share would otherwise be
// computed ahead of them and held (spilled) for all of them.
__device__ __forceinline__ WorkItem opaque(WorkItem it) {
  asm volatile("" : "+s"(it.page_begin), "+s"(it.tok_begin), "+s"(it.tok_count), "+s"(it.first_page), "+s"(it.q_begin), "+s"(it.q_count));
  return it;
}

// ================================================================== 16-row tiles
// Items of at most 16 rows (a sequence alone, few heads a group), and all at head_dim 256,
// where 32-row tiles would not leave two workgroups a CU their registers.  Two waves share
// a row tile's tokens while there are at most two row tiles, each with a softmax of its
// own, joined in LDS at the end; with one row tile the other two take half the output's
// columns (and the same scores).  (16 sequences of up to 6000 tokens: 30 us, bound by the
// codes' bytes.)
template <typename T, int D, int RT, int PG, bool QUADS>
__device__ __forceinline__ void tile_item(const AttnArgs& a, const WorkItem& item, int kvh, TileShared<D>& sh) {
  const WorkItem it = opaque(item);
  constexpr int CPR = D / 16;                        // 16-code chunks of a row
  using Loader = Codes<D, PG, swz<CPR>>;
  constexpr int PLANE = Loader::PLANE, STAGE = Loader::STAGE, NST = TileShared<D>::kStages;
  constexpr int KP = D / 64;                         // K chunk quads: two QK contraction steps each
  constexpr int TS = RT == 4 ? 1 : 2;                // waves sharing a row tile: token halves,
  constexpr int CS = RT == 1 ? 2 : 1;                // and head_dim halves of Oᵀ
  constexpr int NSUB = 4 / TS;                       // 16-token sub-tiles per wave per tile
  constexpr int MT = D / 16 / CS;                    // Oᵀ head_dim tiles of a wave
  constexpr int COMB_SLOT = (MT * 64 * 4 + 2 * 64) * 4;
  static_assert(TS == 1 || 2 * COMB_SLOT <= TileShared<D>::kStages * STAGE, "combine scratch must fit");

  unsigned char* stage = sh.stage;
  int32_t* nan_tok = sh.nan_tok;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int w = rfl(tid >> 6), lane = tid & 63, lg = lane >> 4, lc = lane & 15;
  const int g = a.g, R = it.q_count * g;
  const int n_tiles = (it.tok_count + kTile - 1) / kTile;
  const uint32_t lds0 = lds_addr(stage);
  Loader ld;
  ld.begin(a, it, kvh, tid);

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
  // Q, which left with the page ids, has landed before the tile loads go out: a later
  // first use would make the compiler wait for them too
#pragma unroll
  for (int x = 0; x < 2 * KP; ++x) asm volatile("" : "+v"(qf[x]));
  ld.stage(a, kvh, sh.pg, sh.ks, sh.vs);
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (i < n_tiles) ld.load(lds0 + i * STAGE);
  for (int i = tid; i < D; i += 256) nan_tok[i] = INT32_MAX;
  if (tid == 0) sh.nan_any = 0;
  auto k_scale = [&](int t) { return __uint_as_float(sh.ks[ld.page_of(t)] << 23); };
  auto v_scale = [&](int t) { return __uint_as_float(sh.vs[ld.page_of(t)] << 23); };
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

  int st = 0;
  for (int tile = 0; tile < n_tiles; ++tile, st = st + 1 == NST ? 0 : st + 1) {
    // this wave's loads of the tile have landed (those of the next NST - 2 may be in
    // flight); after the barrier everyone's have, and everyone is done with the tile
    // before, whose stage the tile NST - 1 ahead takes
    if (NST > 2 && tile + 1 < n_tiles) Loader::template wait<1>();
    else Loader::template wait<0>();
    if (tile + NST - 1 < n_tiles) ld.load(lds0 + (st == 0 ? NST - 1 : st - 1) * STAGE);
    if (unseen < min(it.tok_count, (tile + 1) * kTile)) {
      // tokens that a row must not see: their NaN would reach it by a weight of 0
      set_nans_aside<D, swz<CPR>>(stage + st * STAGE + PLANE, tile * kTile, tid, nan_tok, &sh.nan_any);
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
    if (sh.nan_any) {
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

constexpr int kWaveRows = 32;
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ v16f mfma32(v8s a, v8s b, v16f c) {
  if constexpr (std::is_same<T, bf16_t>::value) {
    typedef __bf16 v8b __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  } else {
    typedef _Float16 v8h __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
}

// The value of the lane with the other bit 5 (the other token quads of the same row).
__device__ __forceinline__ float other_half(float x, bool sum) {
  typedef unsigned int u2 __attribute__((ext_vector_type(2)));
  const unsigned xb = __float_as_uint(x);
  const u2 r = __builtin_amdgcn_permlane32_swap(xb, xb, false, false);
  const unsigned a = r.x, b = r.y;
  return sum ? __uint_as_float(a) + __uint_as_float(b) : fmaxf(__uint_as_float(a), __uint_as_float(b));
}

// ================================================================== 32-row tiles
// The same of the 32-row tiles below: 16 consecutive rows' chunk, and the rows 4 h .. + 3
// and 8 + 4 h .. + 3 by two chunks of a half wave's transposed V read.
template <int CPR>
__device__ __forceinline__ int swz32(int r) {
  return CPR == 8 ? ((r >> 1) & 1) << 1 | ((r >> 3) & 1) << 2 | ((r >> 2) & 1) : ((r >> 3) & 1) << 1 | ((r >> 2) & 1);
}

// Items of 17 to 64 rows (a prefix that some beams share), head_dim 64 or 128: RT 32-row
// tiles on v_mfma_f32_32x32x16, so that an operand's conversion serves 32 rows; two
// waves share a row tile's tokens (and with one row tile two its columns).  The C layout
// of a 32-token Sᵀ block (lane l: row l % 32, tokens 8 (i / 4) + 4 (l / 32) + i % 4) is,
// eight registers at a time, the B operand of Oᵀ += Vᵀ Pᵀ over the token order that the
// transposed V reads follow.  The reference of a row's softmax follows its maximum only
// beyond 2^8, so most tiles rescale nothing.  Against 16-row tiles for the same items:
// 4096-token prefixes of 64 rows 203 -> 178 us over four layers.
template <typename T, int D, int RT, int PG, bool QUADS>
__device__ __forceinline__ void tile32_item(const AttnArgs& a, const WorkItem& item, int kvh, TileShared<D>& sh) {
  const WorkItem it = opaque(item);
  constexpr int CPR = D / 16;                        // 16-code chunks of a row
  using Loader = Codes<D, PG, swz32<CPR>>;
  constexpr int PLANE = Loader::PLANE, STAGE = Loader::STAGE, NST = TileShared<D>::kStages;
  constexpr int KP = D / 32;                         // K chunk pairs: two QK contraction steps each
  constexpr int CS = RT == 1 ? 2 : 1;
  constexpr int MB = D / 32 / CS;                    // Oᵀ head_dim blocks of a wave
  constexpr int COMB_SLOT = (MB * 8 * 64 + 2 * 64) * 4;
  // bf16: K's scale in its conversion (every lane holds one token's codes); fp16, whose
  // values it could take out of range, on the fp32 scores
  constexpr bool POST = std::is_same<T, f16_t>::value;
  static_assert(4 * COMB_SLOT <= NST * STAGE, "combine scratch must fit");

  unsigned char* stage = sh.stage;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int w = rfl(tid >> 6), lane = tid & 63, h = lane >> 5, lr = lane & 31;
  const int g = a.g, R = it.q_count * g;
  const int n_tiles = (it.tok_count + kTile - 1) / kTile;
  const uint32_t lds0 = lds_addr(stage);
  Loader ld;
  ld.begin(a, it, kvh, tid);

  // ---- wave role
  const int rt = RT == 1 ? 0 : w & 1, ts = RT == 1 ? w & 1 : w >> 1, cs = RT == 1 ? w >> 1 : 0;
  const bool active = rt * 32 < R;
  const int row = rt * 32 + lr;
  // row / g for row < 256 (the quotient's distance from an integer is at least 1 / (2 g))
  const int j = (int)(((float)row + 0.5f) * (1.f / (float)g)), hh = row - j * g;

  // ---- Q as the B operand: product 2 kp + i takes head_dim 16 (2 kp + h) + 8 i .. + 7
  v8s qf[2 * KP];
  if (row < R) {
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(it.q_begin + j) * a.q_sn + (int64_t)(kvh * g + hh) * a.q_sh;
#pragma unroll
    for (int x = 0; x < 2 * KP; ++x) qf[x] = *reinterpret_cast<const v8s*>(qp + 16 * (2 * (x >> 1) + h) + 8 * (x & 1));
    // (the max is of unscaled scores: a negative scale moves its sign into Q, a zero one zeroes Q)
    if (!POST && a.scale_log2 <= 0.f) {
#pragma unroll
      for (int x = 0; x < 2 * KP; ++x) qf[x] = a.scale_log2 == 0.f ? (v8s)(short)0 : qf[x] ^ (v8s)(short)0x8000;
    }
  } else {
#pragma unroll
    for (int x = 0; x < 2 * KP; ++x) qf[x] = v8s{0, 0, 0, 0, 0, 0, 0, 0};
  }
#pragma unroll
  for (int x = 0; x < 2 * KP; ++x) asm volatile("" : "+v"(qf[x]));
  ld.stage(a, kvh, sh.pg, sh.ks, sh.vs);
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (i < n_tiles) ld.load(lds0 + i * STAGE);
  for (int i = tid; i < D; i += 256) sh.nan_tok[i] = INT32_MAX;
  if (tid == 0) sh.nan_any = 0;
  int lim;
  {
    const int64_t v = (int64_t)it.vis0 + j - it.tok_begin;
    lim = (int)std::min<int64_t>(it.tok_count, std::max<int64_t>(v, 0));
  }
  const int unseen = (int)std::min<int64_t>(it.tok_count, std::max<int64_t>((int64_t)it.vis0 - it.tok_begin, 0));
  // ---- operand offsets (the swizzle repeats every 16 rows, and stages start on 2 KB: the
  // chunks of a row differ by an XOR, which costs an instruction and saves the registers)
  const uint32_t koff = lr * D + ((h ^ swz32<CPR>(lr)) << 4);
  const int vj = (lane & 15) >> 1, vr = (vj >> 2) * 8 + 4 * h + (vj & 3);
  const uint32_t voff = vr * D + (((2 * cs * MB + ((lane >> 4) & 1)) ^ swz32<CPR>(vr)) << 4) + (lane & 1) * 8;

  const float scale = POST || a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
  float m_run = -INFINITY, l_run = 0.f;              // the sums' reference (times `scale`), the weights' sum
  v16f o_acc[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int i = 0; i < 16; ++i) o_acc[mb][i] = 0.f;

  int st = 0;
  for (int tile = 0; tile < n_tiles; ++tile, st = st + 1 == NST ? 0 : st + 1) {
    // (as in the 16-row tiles: this tile has landed, the tile before is done with)
    if (NST > 2 && tile + 1 < n_tiles) Loader::template wait<1>();
    else Loader::template wait<0>();
    if (tile + NST - 1 < n_tiles) ld.load(lds0 + (st == 0 ? NST - 1 : st - 1) * STAGE);
    if (unseen < min(it.tok_count, (tile + 1) * kTile)) {
      set_nans_aside<D, swz32<CPR>>(stage + st * STAGE + PLANE, tile * kTile, tid, sh.nan_tok, &sh.nan_any);
      stream::lds_sync();
    }
    const int s0 = tile * kTile + ts * 32;           // first token of the wave's block
    if (!active || s0 >= it.tok_count) continue;
    const unsigned char* kt = stage + st * STAGE + ts * 32 * D;
    const unsigned char* vt = kt + PLANE;
    // every LDS read of the tile well ahead of its use: K's codes and the scales, then V's
    // codes under the softmax
    v4i kc[KP];
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) kc[kp] = *reinterpret_cast<const v4i*>(kt + (koff ^ (kp << 5)));
    // scales: K of the lane's row, or (POST) K, and V, of its tokens in the C layout,
    // quad 8 i + 4 h .. + 3 or one each
    constexpr int NS = QUADS ? 4 : 16;
    auto token = [&](int i) { return s0 + (QUADS ? 8 * i + 4 * h : 8 * (i >> 2) + 4 * h + (i & 3)); };
    float kr = 1.f, ks[POST ? NS : 1], vs[NS];
    if constexpr (!POST) kr = __uint_as_float(sh.ks[ld.page_of(s0 + lr)] << 23);
    if constexpr (PG == 2) {                         // 16 tokens: one page
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int pg = ld.page_of(s0 + 8 * i);
        if constexpr (POST) ks[i] = ks[i + 1] = __uint_as_float(sh.ks[pg] << 23) * a.scale_log2;
        vs[i] = vs[i + 1] = __uint_as_float(sh.vs[pg] << 23);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int pg = ld.page_of(token(i));
        if constexpr (POST) ks[i] = __uint_as_float(sh.ks[pg] << 23) * a.scale_log2;
        vs[i] = __uint_as_float(sh.vs[pg] << 23);
      }
    }
    v16f x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      x = mfma32<T>(codes8<T>(kc[kp][0], kc[kp][1], kr), qf[2 * kp], x);
      x = mfma32<T>(codes8<T>(kc[kp][2], kc[kp][3], kr), qf[2 * kp + 1], x);
    }
    v2i vc[2][MB];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) vc[s][mb] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i_t)(vt + s * 16 * D + (voff ^ (mb << 5))));
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (POST) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= ks[QUADS ? i >> 2 : i];
    }
    if (__builtin_amdgcn_ballot_w64(lim < s0 + 32) != 0) {
      const int left = lim - s0 - 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i >> 2) + (i & 3) >= left) x[i] = -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    mx = other_half(mx, false) * scale;
    // The reference follows when a row's largest score is 2^8 ahead of it (weights, their
    // sum and Oᵀ are fp32 or of 8 bits' more range): most tiles rescale nothing
    if (__builtin_amdgcn_ballot_w64(mx > m_run + 8.f) != 0) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));   // 0 while nothing was seen
      l_run *= alpha;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o_acc[mb] *= alpha;
      m_run = m_new;
    }
    const float msafe = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t pw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(x[8 * s + 2 * i], scale, -msafe));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(x[8 * s + 2 * i + 1], scale, -msafe));
        l_run += p0 + p1;
        pw[i] = stream::pack2<T>(p0, p1);
      }
      const v8s pf = __builtin_bit_cast(v8s, (u4){pw[0], pw[1], pw[2], pw[3]});
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        u4 vv;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          if constexpr (QUADS) {
            vv[2 * o] = value2<T, false>(vc[s][mb][o], vs[2 * s + o]);
            vv[2 * o + 1] = value2<T, true>(vc[s][mb][o], vs[2 * s + o]);
          } else {
            vv[2 * o] = value11<T, false>(vc[s][mb][o], vs[8 * s + 4 * o], vs[8 * s + 4 * o + 1]);
            vv[2 * o + 1] = value11<T, true>(vc[s][mb][o], vs[8 * s + 4 * o + 2], vs[8 * s + 4 * o + 3]);
          }
        }
        o_acc[mb] = mfma32<T>(__builtin_bit_cast(v8s, vv), pf, o_acc[mb]);
      }
    }
  }
  l_run = other_half(l_run, true);

  // ---- the two token halves exchange half of their columns and each finishes its own
  const int pair = RT == 1 ? cs : rt;
  float* give = reinterpret_cast<float*>(stage) + (2 * pair + ts) * (COMB_SLOT / 4);
  const float* take = reinterpret_cast<const float*>(stage) + (2 * pair + (ts ^ 1)) * (COMB_SLOT / 4);
  constexpr int HB = MB * 4 / 2;                     // v4f groups (mb, i) of a half
  auto group = [&](int q) { return v4f{o_acc[q >> 2][4 * (q & 3)], o_acc[q >> 2][4 * (q & 3) + 1], o_acc[q >> 2][4 * (q & 3) + 2], o_acc[q >> 2][4 * (q & 3) + 3]}; };
  __syncthreads();                                   // tiles no longer needed
  if (active) {
#pragma unroll
    for (int q = 0; q < HB; ++q) *reinterpret_cast<v4f*>(give + (q * 64 + lane) * 4) = ts ? group(q) : group(HB + q);
    give[HB * 256 + lane] = m_run;
    give[HB * 256 + 64 + lane] = l_run;
  }
  __syncthreads();
  if (!active) return;
  const float mb_ = take[HB * 256 + lane], lb = take[HB * 256 + 64 + lane];
  const float M = fmaxf(m_run, mb_);
  const float ca = (M == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(m_run - M);
  const float cb = (M == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(mb_ - M);
  l_run = l_run * ca + lb * cb;
  const float inv = l_run > 0.f ? 1.f / l_run : 0.f, fa = ca * inv, fb = cb * inv;
  v4f y[HB];
#pragma unroll
  for (int q = 0; q < HB; ++q) {
    const v4f v = *reinterpret_cast<const v4f*>(take + (q * 64 + lane) * 4), mine = ts ? group(HB + q) : group(q);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[q][e] = fmaf(v[e], fb, mine[e] * fa);
  }
  // lane holds Oᵀ[d0 + 32 (q / 4) + 8 (q % 4) .. + 3][row] (the row's query and head again,
  // not held in registers through the tiles)
  int row_ = row;
  asm volatile("" : "+v"(row_));
  const int j_ = (int)(((float)row_ + 0.5f) * (1.f / (float)g)), head = kvh * g + row_ - j_ * g;
  const int d0 = 32 * cs * MB + (ts * HB / 4) * 32 + 4 * h;
  static_assert(HB % 4 == 0 || MB == 1, "a half is whole blocks, or half of one");
  const int q0 = MB == 1 ? ts * HB : 0;              // (one block: the half's first quad)
  if (sh.nan_any) {
#pragma unroll
    for (int q = 0; q < HB; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (sh.nan_tok[d0 + 32 * (q >> 2) + 8 * ((q0 + q) & 3) + e] < lim) y[q][e] = NAN;
  }
  if (row_ >= R) return;
  if (it.out_row < 0) {
    T* op = reinterpret_cast<T*>(a.out) + (int64_t)(it.q_begin + j_) * a.o_sn + (int64_t)head * a.o_sh + d0;
#pragma unroll
    for (int q = 0; q < HB; ++q) *reinterpret_cast<v4s*>(op + 32 * (q >> 2) + 8 * ((q0 + q) & 3)) = pack4<T>(y[q][0], y[q][1], y[q][2], y[q][3]);
  } else {
    float* op = a.part_o + ((int64_t)(it.out_row + j_) * a.hq + head) * D + d0;
#pragma unroll
    for (int q = 0; q < HB; ++q) *reinterpret_cast<v4f*>(op + 32 * (q >> 2) + 8 * ((q0 + q) & 3)) = y[q];
  }
  if (h == 0 && cs == 0 && ts == 0) store_lse(a, it, j_, head, M, l_run);
}

// ================================================================== one wave an item
// Short items of at most 16 rows (a beam's own tokens), pages of a multiple of 16 tokens:
// each wave of a workgroup takes an item of its own, in steps of 16 tokens through its
// share of the stages (as many steps in flight as the others have tiles), with no barrier.
// Four such items would otherwise be four workgroups that start, wait and end for a tile
// or two each: 8 x 16 beams with tails of up to 24 tokens 200 -> 186 us over 8 layers.
// All of a step's tokens lie in one page, so its scales are scalars.
template <typename T, int D>
__device__ __forceinline__ void wave_item(const AttnArgs& a, const WorkItem& item, int kvh, TileShared<D>& sh, int w) {
  const WorkItem it = opaque(item);
  constexpr int CPR = D / 16, RPI = 64 / CPR, IPW = 16 / RPI, NST = TileShared<D>::kStages;
  constexpr int PLANE = 16 * D, STEP = 2 * PLANE, OPS = 2 * IPW;
  constexpr int KP = D / 64, MT = D / 16;
  const int lane = threadIdx.x & 63, lg = lane >> 4, lc = lane & 15;
  const int g = a.g, R = it.q_count * g, ps = a.page_size;
  unsigned char* ring = sh.stage + w * NST * STEP;
  const uint32_t lds0 = lds_addr(ring);

  // ---- page ids (with Q), then scales and the first steps
  const int slot0 = it.tok_begin - it.first_page * ps;
  const int n_pages = (int)(((float)(slot0 + it.tok_count - 1) + 0.5f) * (1.f / (float)ps)) + 1;
  const int id = a.pages[it.page_begin + it.first_page + min(lane, n_pages - 1)];
  const int row = lc, j = (int)(((float)row + 0.5f) * (1.f / (float)g)), hh = row - j * g;
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
  const uint8_t* sp = a.kv_scale + (int64_t)id * 2 * a.hkv + kvh;
  const int k_byte = sp[0], v_byte = sp[a.hkv];
  const uint32_t row_bytes = (uint32_t)a.hkv * D, vplane = (uint32_t)ps * row_bytes, page_bytes = 2 * vplane;
  const uint64_t kvb = reinterpret_cast<uint64_t>(a.kv) + (uint64_t)kvh * D;
  uint32_t off[IPW];
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const int r = i * RPI + lane / CPR;
    off[i] = (uint32_t)r * row_bytes + ((uint32_t)((lane % CPR) ^ swz<CPR>(r)) << 4);
  }
  const int steps = (it.tok_count + 15) >> 4;
  int l_page = 0, l_slot = slot0, l_tok = 0;           // of the next step to load
  auto load = [&](uint32_t dst) {
    const uint32_t pid = (uint32_t)__builtin_amdgcn_readlane(id, l_page);
    const uint64_t base = kvb + (uint64_t)pid * page_bytes + (uint32_t)l_slot * row_bytes;
    const int left = it.tok_count - 1 - l_tok;         // rows of this step up to the item's last token
    if (left >= 15) {
#pragma unroll
      for (int i = 0; i < IPW; ++i) dma16_s(base, off[i], dst + i * 1024);
#pragma unroll
      for (int i = 0; i < IPW; ++i) dma16_s(base + vplane, off[i], dst + PLANE + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < IPW; ++i) {
        const int r = i * RPI + lane / CPR;
        const uint64_t src = base + (uint32_t)min(r, left) * row_bytes + ((uint32_t)((lane % CPR) ^ swz<CPR>(r)) << 4);
        stream::dma16(reinterpret_cast<const void*>(src), dst + i * 1024);
        stream::dma16(r <= left ? reinterpret_cast<const void*>(src + vplane) : &kZeroChunk, dst + PLANE + i * 1024);
      }
    }
    l_tok += 16;
    l_slot += 16;
    if (l_slot >= ps) {
      l_slot -= ps;
      ++l_page;
    }
  };
#pragma unroll
  for (int i = 0; i < NST; ++i)
    if (i < steps) load(lds0 + i * STEP);

  // ---- operand offsets
  uint32_t koff[KP];
#pragma unroll
  for (int kp = 0; kp < KP; ++kp) koff[kp] = lc * D + (((4 * kp + lg) ^ swz<CPR>(lc)) << 4);
  const int vr = 4 * lg + ((lc >> 1) & 3);             // (a transposed read takes 8 rows: these four, twice)
  float m_run = -INFINITY, l_run = 0.f;
  v4f o_acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) o_acc[mt] = v4f{0.f, 0.f, 0.f, 0.f};
  int page = 0, slot = slot0, st = 0;
  for (int step = 0; step < steps; ++step, st = st + 1 == NST ? 0 : st + 1) {
    // this step's loads have landed, those of up to NST - 1 newer ones may be in flight
    const int newer = min(NST - 1, steps - 1 - step);
    if (newer == 0) __builtin_amdgcn_s_waitcnt(BE_VMCNT(0));
    else if (newer == 1) __builtin_amdgcn_s_waitcnt(BE_VMCNT(OPS));
    else __builtin_amdgcn_s_waitcnt(BE_VMCNT(2 * OPS));
    asm volatile("" ::: "memory");
    const unsigned char* kt = ring + st * STEP;
    const unsigned char* vt = kt + PLANE;
    const float ks = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(k_byte, page) << 23) * a.scale_log2;
    const float vs = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(v_byte, page) << 23);
    slot += 16;
    if (slot >= ps) {
      slot -= ps;
      ++page;
    }
    v4i kc[KP];
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) kc[kp] = *reinterpret_cast<const v4i*>(kt + koff[kp]);
    v2i vc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      vc[mt] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i_t)(vt + vr * D + ((mt ^ swz<CPR>(vr)) << 4) + (lc & 1) * 8));
    v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      x = mfma_qk<T>(codes8<T>(kc[kp][0], kc[kp][1]), qf[2 * kp], x);
      x = mfma_qk<T>(codes8<T>(kc[kp][2], kc[kp][3]), qf[2 * kp + 1], x);
    }
    x *= ks;
    const int left = it.tok_count - step * 16 - 4 * lg;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r >= left) x[r] = -INFINITY;
    const float mx = rows4_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    if (__builtin_amdgcn_ballot_w64(mx > m_run + 8.f) != 0) {         // (as in the 32-row tiles)
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      l_run *= alpha;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o_acc[mt] *= alpha;
      m_run = m_new;
    }
    const float msafe = m_run == -INFINITY ? 0.f : m_run;
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      p[r] = __builtin_amdgcn_exp2f(x[r] - msafe);
      l_run += p[r];
    }
    const v4s pf = pack4<T>(p[0], p[1], p[2], p[3]);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
      o_acc[mt] = mfma_pv<T>(__builtin_bit_cast(v4s, (u2){value2<T, false>(vc[mt][0], vs), value2<T, true>(vc[mt][0], vs)}), pf, o_acc[mt]);
    }
    if (step + NST < steps) {
      __builtin_amdgcn_s_waitcnt(0xc07f);              // lgkmcnt(0): this step's reads are done with its stage
      load(lds0 + st * STEP);
    }
  }
  l_run = rows4_sum(l_run);
  if (row >= R) return;
  const int head = kvh * g + hh;
  const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
  if (it.out_row < 0) {
    T* op = reinterpret_cast<T*>(a.out) + (int64_t)(it.q_begin + j) * a.o_sn + (int64_t)head * a.o_sh;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      *reinterpret_cast<v4s*>(op + mt * 16 + 4 * lg) =
          pack4<T>(o_acc[mt][0] * inv, o_acc[mt][1] * inv, o_acc[mt][2] * inv, o_acc[mt][3] * inv);
  } else {
    float* op = a.part_o + ((int64_t)(it.out_row + j) * a.hq + head) * D;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<v4f*>(op + mt * 16 + 4 * lg) = o_acc[mt] * inv;
  }
  if (lg == 0) store_lse(a, it, j, head, m_run, l_run);
}

// A workgroup takes as many row tiles as its item has: with fewer, the waves share out
// the tokens of a row tile (and the columns) rather than idle.
template <typename T, int D, int PG, bool QUADS>
__global__ __launch_bounds__(256, D == 256 || !QUADS ? 2 : D == 128 ? 3 : 4) void attn_kv8_kernel(AttnArgs a, int first_item, int end_item, int waves) {
  __shared__ __attribute__((aligned(1024))) TileShared<D> sh;
  // items [first, end - waves) by workgroups, the last `waves` by one wave each
  if (a.live_blocks) {
    first_item = a.live_blocks[0];
    waves = a.live_blocks[kHdrWaves - kHdrBlocks];
    end_item = *a.live_items;
  }
  const int wg = item_of(a, blockIdx.x), kvh = (int)blockIdx.x - wg * a.hkv, item = first_item + wg, singles = end_item - waves;
  if (item >= singles) {
    if constexpr (PG == 2) {
      const int w = rfl(threadIdx.x >> 6), mine = singles + 4 * (item - singles) + w;
      if (mine < end_item) wave_item<T, D>(a, item_at(a, mine), kvh, sh, w);
    }
    return;
  }
  const WorkItem it = item_at(a, rfl(item));
  const int R = it.q_count * a.g;
  if (R <= 16) {
    tile_item<T, D, 1, PG, QUADS>(a, it, kvh, sh);
  } else if constexpr (D == 256) {                   // (32-row tiles would not fit the registers)
    if (R <= 32) tile_item<T, D, 2, PG, QUADS>(a, it, kvh, sh);
    else tile_item<T, D, 4, PG, QUADS>(a, it, kvh, sh);
  } else {
    if (R <= 32) tile32_item<T, D, 1, PG, QUADS>(a, it, kvh, sh);
    else tile32_item<T, D, 2, PG, QUADS>(a, it, kvh, sh);
  }
}

template <typename T, int D>
static int launch_tile(const be_attn_plan_info* info, const AttnArgs& a, hipStream_t st) {
  const int first = info->num_wg;                    // the block kernel's items come first
  const int end = info->grid_items, waves = info->num_tail_items;
  const unsigned grid = (unsigned)(info->static_layout ? end : end - first - waves + (waves + 3) / 4) * info->num_kv_heads;
  if (grid == 0) return BE_OK;
  if (a.page_size % 16 == 0) attn_kv8_kernel<T, D, 2, true><<<grid, 256, 0, st>>>(a, first, end, waves);
  else if (paged4(a.page_size, D)) attn_kv8_kernel<T, D, 1, true><<<grid, 256, 0, st>>>(a, first, end, waves);
  else if (a.page_size % 4 == 0) attn_kv8_kernel<T, D, 0, true><<<grid, 256, 0, st>>>(a, first, end, waves);
  else attn_kv8_kernel<T, D, 0, false><<<grid, 256, 0, st>>>(a, first, end, waves);
  BE_HIP_CHECK(hipGetLastError());
  return BE_OK;
}

// ================================================================== 128-row blocks
// The 16-byte chunk XOR of a row of 16-bit values: any 16 consecutive rows' chunk and
// the four rows x four chunks of a half wave's transposed V read fall on all banks.
template <int D>
__device__ __forceinline__ int swz16(int r) {
  return D == 128 ? ((r & 3) << 2 | ((r >> 2) & 3)) : (((r >> 1) & 1) << 2 | ((r >> 2) & 3));
}

// Groups whose query tiles have 65 to 128 rows (prompts, prefixes that many beams share),
// head_dim 64 or 128:
// one workgroup of four waves, 32 rows each, over 64-token tiles, products on
// v_mfma_f32_32x32x16.  At this many rows an operand is read by every wave, so a tile
// is turned into 16-bit values once, on its way into LDS: each thread loads its share
// of the next tile's codes into registers while the current one is computed, converts
// it and writes it to the other stage; one barrier a tile.  K is converted relative to
// the item's largest K scale, which the softmax's scale takes back.  8 prompts of 1024
// tokens, 32 heads of 128 over 8: 102 us, 670 TFLOP/s with the masked halves of the
// diagonal tiles as work not done (the tiles above take 107 to 111 for the same); bound by the
// matrix instructions' waits for LDS and for the next tile's conversion.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void attn_kv8_block_kernel(AttnArgs a, int n_items) {
  constexpr int KS = D / 16;                         // QK contraction steps
  constexpr int MB = D / 32;                         // Oᵀ head_dim blocks
  constexpr int RB = D * 2, PLANE = kTile * RB, STAGE = 2 * PLANE;
  constexpr int CPR = D / 16;                        // 16-code chunks of a row
  constexpr int NC = kTile * CPR / 256;              // K (and V) chunks of a thread
  constexpr int CPR16 = D / 8, RPI = 64 / CPR16;     // of the 16-bit rows

  __shared__ __attribute__((aligned(1024))) unsigned char stage[2 * STAGE];
  __shared__ int32_t pg_lds[kMaxPagesKv8];
  __shared__ uint16_t sc_lds[kMaxPagesKv8];          // scale bytes of the pages: K | V << 8
  __shared__ int32_t nan_tok[D];
  __shared__ int32_t nan_any, k_top;
  const int item = item_of(a, blockIdx.x), kvh = (int)blockIdx.x - item * a.hkv;
  if (item >= (a.live_blocks ? *a.live_blocks : n_items)) return;

  const WorkItem it = item_at(a, item);
  const int tid = threadIdx.x;
  const int w = rfl(tid >> 6), lane = tid & 63, h = lane >> 5, lr = lane & 31;
  const int g = a.g, R = it.q_count * g, ps = a.page_size;

  // ---- the item's pages and their scales
  const int first_page = it.first_page;
  const float inv_ps = 1.f / (float)ps;
  const int slot0 = it.tok_begin - first_page * ps;
  const int n_pages = (int)(((float)(slot0 + it.tok_count - 1) + 0.5f) * inv_ps) + 1;
  const int n_tiles = (it.tok_count + kTile - 1) / kTile;
  if (tid == 0) {
    nan_any = 0;
    k_top = 0;
  }
  for (int i = tid; i < D; i += 256) nan_tok[i] = INT32_MAX;
  __syncthreads();
  {
    int top = 0;
    for (int i = tid; i < n_pages; i += 256) {
      const int id = a.pages[it.page_begin + first_page + i];
      const int64_t at = (int64_t)id * 2 * a.hkv + kvh;
      const int kb = a.kv_scale[at], vb = a.kv_scale[at + a.hkv];
      pg_lds[i] = id;
      sc_lds[i] = (uint16_t)(kb | vb << 8);
      top = max(top, kb);
    }
    if (top > 0) atomicMax(&k_top, top);
  }

  // ---- this wave's rows: lane's row, the tokens it sees, the wave's most
  const int row = w * kWaveRows + lr;
  const bool wave_on = w * kWaveRows < R;
  const float inv_g = 1.f / (float)g;
  // row / g for row < 256 (the quotient's distance from an integer is at least 1 / (2 g))
  auto query_of = [&](int r) { return (int)(((float)r + 0.5f) * inv_g); };
  int lim;
  {
    const int64_t v = (int64_t)it.vis0 + query_of(min(row, R - 1)) - it.tok_begin;
    lim = (int)std::min<int64_t>(it.tok_count, std::max<int64_t>(v, 0));
  }
  const int lim_most = __builtin_amdgcn_readlane(lim, 31);   // rows are in query order
  const int unseen = (int)std::min<int64_t>(it.tok_count, std::max<int64_t>((int64_t)it.vis0 - it.tok_begin, 0));

  // ---- Q as the B operand: lane holds Q[row][16 ks + 8 h .. +7]; a negative scale moves
  // its sign into Q, a zero one zeroes Q (the softmax takes the max of unscaled scores)
  v8s qf[KS];
  if (row < R) {
    const int j = query_of(row), hh = row - j * g;
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(it.q_begin + j) * a.q_sn + (int64_t)(kvh * g + hh) * a.q_sh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const v8s*>(qp + ks * 16 + h * 8);
    if (a.scale_log2 <= 0.f) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = a.scale_log2 == 0.f ? (v8s)(short)0 : qf[ks] ^ (v8s)(short)0x8000;
    }
  } else {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = v8s{0, 0, 0, 0, 0, 0, 0, 0};
  }
  __syncthreads();                                   // page ids and scales staged
  const int k_ref = max(k_top, 27);                  // (27: the least exponent; pages not written have byte 0)
  const float scale = (a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2)) * __uint_as_float((uint32_t)k_ref << 23);

  // ---- tile loads: thread's chunks tid + 256 i of K and of V
  const uint32_t row_bytes = (uint32_t)a.hkv * D;
  const uint8_t* kv = reinterpret_cast<const uint8_t*>(a.kv) + (int64_t)kvh * D;
  v4i kc[NC], vc[NC];
  int sc[NC];
  auto fetch = [&](int tile) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = tid + 256 * i, t = tile * kTile + c / CPR;
      kc[i] = vc[i] = v4i{0, 0, 0, 0};               // (past the end: scores are masked, V is zeros)
      sc[i] = 0;
      if (t < it.tok_count) {
        const int pi = (int)(((float)(slot0 + t) + 0.5f) * inv_ps), sl = slot0 + t - pi * ps;
        sc[i] = sc_lds[pi];
        const uint8_t* src = kv + ((uint64_t)((uint32_t)pg_lds[pi] * 2u) * (uint32_t)ps + (uint32_t)sl) * row_bytes + (c % CPR) * 16;
        kc[i] = *reinterpret_cast<const v4i*>(src);
        vc[i] = *reinterpret_cast<const v4i*>(src + (uint64_t)ps * row_bytes);
      }
    }
  };
  auto put = [&](int tile, unsigned char* to) {
    const bool masked = unseen < min(it.tok_count, (tile + 1) * kTile);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = tid + 256 * i, r = c / CPR, ch = (c % CPR) * 2;
      if (masked && __builtin_expect((nan_bytes(vc[i][0]) | nan_bytes(vc[i][1]) | nan_bytes(vc[i][2]) | nan_bytes(vc[i][3])) != 0, 0)) {
        // tokens that a row must not see: their NaN would reach it by a weight of 0
#pragma unroll
        for (int b = 0; b < 16; ++b)
          if (((vc[i][b >> 2] >> (8 * (b & 3))) & 0x7f) == 0x7f) {
            atomicMin(&nan_tok[(c % CPR) * 16 + b], tile * kTile + r);
            vc[i][b >> 2] &= ~(0xff << (8 * (b & 3)));
          }
        nan_any = 1;
      }
      const float ks = __uint_as_float((uint32_t)max((sc[i] & 0xff) - k_ref + 127, 0) << 23), vs = __uint_as_float((uint32_t)(sc[i] >> 8) << 23);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t at = r * RB + (((ch + half) ^ swz16<D>(r)) << 4);
        *reinterpret_cast<u4*>(to + at) = u4{value2<T, false>(kc[i][2 * half], ks), value2<T, true>(kc[i][2 * half], ks),
                                             value2<T, false>(kc[i][2 * half + 1], ks), value2<T, true>(kc[i][2 * half + 1], ks)};
        *reinterpret_cast<u4*>(to + PLANE + at) = u4{value2<T, false>(vc[i][2 * half], vs), value2<T, true>(vc[i][2 * half], vs),
                                                     value2<T, false>(vc[i][2 * half + 1], vs), value2<T, true>(vc[i][2 * half + 1], vs)};
      }
    }
  };

  // ---- operand offsets
  const int r16 = lane & 15, q4 = r16 >> 2, e4 = ((lane >> 4) & 1) * 2 + ((r16 & 3) >> 1);
  uint32_t koff[KS], voff[MB][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = lr * RB + (((2 * ks + h) ^ swz16<D>(lr)) << 4);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int vr = 8 * u + 4 * h + q4;             // the row's low four bits
      voff[mb][u] = vr * RB + (((mb * 4 + e4) ^ swz16<D>(vr)) << 4) + (r16 & 1) * 8;
    }

  // reference of the sums, the largest score (both times `scale`), the weights' sum
  float m_run = -INFINITY, m_top = -INFINITY, l_run = 0.f;
  v16f o_acc[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int i = 0; i < 16; ++i) o_acc[mb][i] = 0.f;

  fetch(0);
  put(0, stage);
  if (n_tiles > 1) fetch(1);
  for (int tile = 0; tile < n_tiles; ++tile) {
    const int st = tile & 1;
    stream::lds_sync();                              // the tile is in its stage, and everyone is done with the other
    const int t0 = tile * kTile;
    const unsigned char* kt = stage + st * STAGE;
    const unsigned char* vt = kt + PLANE;
    // the first K fragments leave LDS while the next tile is converted
    v8s kf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = *reinterpret_cast<const v8s*>(kt + koff[ks]);
    if (tile + 1 < n_tiles) {
      put(tile + 1, stage + (st ^ 1) * STAGE);
      if (tile + 2 < n_tiles) fetch(tile + 2);
    }
    if (!wave_on || t0 >= lim_most) continue;

    v16f x[2];
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[tb][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) x[0] = mfma32<T>(kf[ks], qf[ks], x[0]);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = *reinterpret_cast<const v8s*>(kt + 32 * RB + koff[ks]);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) x[1] = mfma32<T>(kf[ks], qf[ks], x[1]);
    if (__builtin_amdgcn_ballot_w64(lim < t0 + kTile) != 0) {
      const int left = lim - t0 - 4 * h;
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (tb * 32 + 8 * (i >> 2) + (i & 3) >= left) x[tb][i] = -INFINITY;
    }
    // (maximum rather than fmax: a NaN score makes the row NaN either way)
    float top = -INFINITY;
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int i = 0; i < 16; i += 2)
        top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[tb][i], x[tb][i + 1]), top);
    // When a row's largest score grows, every row of the wave takes the tile's largest as
    // its reference, unless it lies 2^8 below the row's: that weight is exact in 16 bits
    top = other_half(top, false) * scale;
    if (__builtin_amdgcn_ballot_w64(top > m_top) != 0) {
      m_top = fmaxf(m_top, top);
      const float m_new = top >= m_top - 8.f ? top : m_run;
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      l_run *= alpha;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o_acc[mb] *= alpha;
      m_run = m_new;
    }
    const float msafe = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v4s vf[MB][2];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          vf[mb][u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((stream::lds_v4s_t)(vt + s * 16 * RB + voff[mb][u]));
      uint32_t pw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(x[s >> 1][8 * (s & 1) + 2 * j], scale, -msafe));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(x[s >> 1][8 * (s & 1) + 2 * j + 1], scale, -msafe));
        l_run += p0 + p1;
        pw[j] = stream::pack2<T>(p0, p1);
      }
      const v8s pf = __builtin_bit_cast(v8s, (u4){pw[0], pw[1], pw[2], pw[3]});
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
        o_acc[mb] = mfma32<T>(__builtin_shufflevector(vf[mb][0], vf[mb][1], 0, 1, 2, 3, 4, 5, 6, 7), pf, o_acc[mb]);
    }
  }

  // ---- writes: lane holds Oᵀ[32 mb + 8 (i / 4) + 4 h + i % 4][row]
  l_run = other_half(l_run, true);
  const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
  const int j = query_of(row), hh = row - j * g, head = kvh * g + hh;
  __syncthreads();                                   // every wave is done with the stages
  if (nan_any) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (nan_tok[32 * mb + 8 * (i >> 2) + 4 * h + (i & 3)] < lim) o_acc[mb][i] = NAN;
  }
  if (it.out_row < 0) {
    // through LDS (the wave's own 32 rows, chunks swizzled by row), so that the stores
    // are whole rows, 16 bytes a lane
    unsigned char* ol = stage + w * kWaveRows * RB;
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const u2 pk = {stream::pack2<T>(o_acc[mb][4 * b] * inv, o_acc[mb][4 * b + 1] * inv),
                       stream::pack2<T>(o_acc[mb][4 * b + 2] * inv, o_acc[mb][4 * b + 3] * inv)};
        *reinterpret_cast<u2*>(ol + lr * RB + (((mb * 4 + b) ^ swz16<D>(lr)) << 4) + 8 * h) = pk;
      }
    // (a wave reads only what it wrote: the compiler's lgkmcnt waits order it)
#pragma unroll
    for (int i = 0; i < kWaveRows / RPI; ++i) {
      const int lrow = i * RPI + lane / CPR16, orow = w * kWaveRows + lrow;
      const uint4 v = *reinterpret_cast<const uint4*>(ol + lrow * RB + (((lane % CPR16) ^ swz16<D>(lrow)) << 4));
      if (orow < R) {
        const int oj = query_of(orow), oh = kvh * g + (orow - oj * g);
        T* op = reinterpret_cast<T*>(a.out) + (int64_t)(it.q_begin + oj) * a.o_sn + (int64_t)oh * a.o_sh;
        *reinterpret_cast<uint4*>(op + (lane % CPR16) * 8) = v;
      }
    }
  } else if (row < R) {
    float* op = a.part_o + ((int64_t)(it.out_row + j) * a.hq + head) * D;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const v4f v = {o_acc[mb][4 * b] * inv, o_acc[mb][4 * b + 1] * inv, o_acc[mb][4 * b + 2] * inv,
                       o_acc[mb][4 * b + 3] * inv};
        *reinterpret_cast<v4f*>(op + mb * 32 + 8 * b + 4 * h) = v;
      }
  }
  if (row < R && h == 0) store_lse(a, it, j, head, m_run, l_run);
}

template <typename T, int D>
static int launch_block(const be_attn_plan_info* info, const AttnArgs& a, hipStream_t st) {
  const int n = info->num_wg;
  if (n == 0) return BE_OK;
  attn_kv8_block_kernel<T, D><<<(unsigned)n * (unsigned)info->num_kv_heads, 256, 0, st>>>(a, n);
  BE_HIP_CHECK(hipGetLastError());
  return BE_OK;
}

template <typename T>
static int launch_d(const be_attn_plan_info* info, const AttnArgs& a, hipStream_t st) {
  if (info->num_wg < 0 || info->num_wg > info->grid_items || (info->num_wg > 0 && info->head_dim == 256))
    return fail(BE_ERR_INVALID, "corrupt plan: %d block items of %d at head_dim %d", info->num_wg, info->grid_items, info->head_dim);
  switch (info->head_dim) {
    case 64:
      if (const int rc = launch_block<T, 64>(info, a, st)) return rc;
      return launch_tile<T, 64>(info, a, st);
    case 128:
      if (const int rc = launch_block<T, 128>(info, a, st)) return rc;
      return launch_tile<T, 128>(info, a, st);
    case 256: return launch_tile<T, 256>(info, a, st);
    default: return fail(BE_ERR_UNSUPPORTED, "head_dim %d", info->head_dim);
  }
}

}  // namespace kv8

int kv8_launch(const be_attn_plan_info* info, const AttnArgs& a, hipStream_t st) {
  return info->dtype == BE_BF16 ? kv8::launch_d<bf16_t>(info, a, st) : kv8::launch_d<f16_t>(info, a, st);
}

}  // namespace be
