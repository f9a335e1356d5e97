// Writes to a paged KV cache held in 8 bits (gfx950): rotary embedding, quantisation
// and append in one launch, page fork copies, and reading the values back.
//
// A layer holds e4m3 codes [num_pages, 2, page_size, num_kv_heads, head_dim] and, for
// each block (the tokens of one page, K or V, one head), a power-of-two scale as an
// e8m0 byte [num_pages, 2, num_kv_heads]: a code c stands for c 2^(byte - 127).  A
// block's exponent E is the least with amax <= 448 2^E (448: the largest code), at
// least kLeastExp.  e4m3 carries an exponent of its own, so a power of two costs no
// precision against a free scale (a value's relative error is at most 2^-4 down to
// 2^-14 of the block's largest), and a stored value is exact in bf16 and, down to its
// subnormal step of 2^-24, in fp16.

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace be {
namespace kv8 {

constexpr int kLeastExp = -100;        // (2^126 of its inverse stays finite)
constexpr int kChunk = 16;             // entries of a workgroup, at most
constexpr int kTile = 256;             // entries of a scan step, members of a batch beyond the chunk's
constexpr int kMembers = kChunk + kTile;
constexpr int kFew = 256;              // entries of a call that takes four a workgroup, at most (a scan step)
constexpr int kFewPages = 4;           // led pages that are looked for one by one
constexpr int kHeads = 4;               // KV heads of a pass, at most

// The largest e4m3 value times a power of two that the type holds: stored values
// saturate there, so that a dequantised value is never an infinity.
template <typename T> __device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<f16_t>() { return 61440.f; }
template <> __device__ __forceinline__ float largest<bf16_t>() { return __uint_as_float(0x7f700000u); }   // 1.875 2^127

// The least E >= kLeastExp with amax <= 448 2^E for the bits of a finite amax >= 0:
// 448 is 1.75 2^8, and a mantissa beyond 1.75 carries into the exponent.
__device__ __forceinline__ int block_exp(uint32_t amax_bits) {
  return max((int)((amax_bits + 0x1fffffu) >> 23) - 127 - 8, kLeastExp);
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // e in [-126, 127]

// Four floats as e4m3 codes (round to nearest, ties to even; NaN and infinities NaN).
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// The largest of 16 lanes (a DPP row), in all of them, by rotations of the row.
template <int N> __device__ __forceinline__ float row_ror(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float max16(float x) {
  x = fmaxf(x, row_ror<8>(x));
  x = fmaxf(x, row_ror<4>(x));
  x = fmaxf(x, row_ror<2>(x));
  return fmaxf(x, row_ror<1>(x));
}

struct AppendArgs {
  const void *q, *k, *v;               // rows of head_dim elements, 16-byte aligned; q: with cos only
  int64_t q_sn, k_sn, k_sh, v_sn, v_sh;
  const void *cos_t, *sin_t;           // [max_pos, head_dim], null: no rotation and no q
  const int64_t* positions;
  void* q_out;                         // [n, hq, head_dim]
  uint8_t *kv, *scale;
  const int32_t *page_idx, *slot;
  int32_t* err;
  int n, hq, hkv, num_pages, page_size, max_pos;
  int hq_share, hkv_share;             // heads of a workgroup
};

// One row of a head over 16 lanes: lane u holds elements u E .. + E - 1 of each half,
// E = D / 32, in v[0..E) and v[E..2E).
template <typename T, int E> struct alignas(2 * E) Pack { T x[E]; };
template <typename T, int E>
__device__ __forceinline__ void unpack(const Pack<T, E>& p, float (&v)[2 * E], int at) {
#pragma unroll
  for (int e = 0; e < E; ++e) v[at + e] = to_f32(p.x[e]);
}
template <typename T, int E>
__device__ __forceinline__ void load_half(const T* p, float (&v)[2 * E], int at) {
  unpack<T, E>(*reinterpret_cast<const Pack<T, E>*>(p), v, at);
}

// HF's rotate_half form in fp32: each product and the sum rounded on its own, so that
// the result does not depend on which the compiler fuses.
template <int E>
__device__ __forceinline__ void rotate(float (&v)[2 * E], const float (&c)[2 * E], const float (&s)[2 * E]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float lo = v[e], hi = v[E + e];
    const float a = lo * c[e], b = -hi * s[e], x = hi * c[E + e], y = lo * s[E + e];
    v[e] = a + b;
    v[E + e] = x + y;
  }
}

// One workgroup takes `chunk` consecutive entries (blockIdx.x) and a share of the
// heads (blockIdx.y of gridDim.y): it rotates the entries' q rows, and it writes the
// K and V of every page that is first named by one of its entries -- all of the call's
// entries of that page, wherever they stand, since they share the block's scale.  The
// other pages of its entries belong to an earlier workgroup.  So each block has one
// writer, in any order of entries, and the stored bytes do not depend on scheduling.
//
// Per page and head: s0 is the least slot the call writes.  s0 = 0 starts the block
// anew; otherwise its exponent only grows, and the s0 tokens before are rescaled by the
// difference (a power of two: exact but for subnormal codes).  The tokens of a page
// are its slots up to the last written one; what lay behind is void.
//
// What bounds it: a decode step's launch is a chain of round trips (indices and rows,
// tables, the old scale): 8.7 us for 128 tokens of 32 heads of 128 over 8; prompts are
// bound by the rows' bytes: 8 x 1024 tokens in 47 to 52 us, 3.9 TB/s with the q rows where a
// copy moves 4.9.  Between them a launch has too few workgroups to hide its chain: 2643
// tokens of 16 heads of 64 over 4, five prompts on pages of 8, 15 us.  The scan of all
// page ids for entries of the same pages is what one writer a block costs: every
// workgroup reads 4 bytes an entry of the call, from L2.
template <typename T, int D, int PER>
__global__ __launch_bounds__(256, D == 64 ? 4 : D == 128 ? 3 : 2) void append_kernel(AppendArgs a) {
  constexpr int E = D / 32;
  __shared__ int32_t s_page[kChunk], s_slot[kChunk], s_lead[kChunk];   // the chunk's pages (-1: skipped), slots, which lead
  __shared__ bool s_dead[kChunk];                         // written again by a later entry of the chunk
  __shared__ int32_t s_first[kChunk];                     // per led page: least slot written
  __shared__ uint32_t s_amax[kHeads][kChunk][2];          // per head, led page, K / V: bits of the largest finite |x|
  __shared__ int32_t s_exp[kHeads][kChunk][2], s_old[kHeads][kChunk][2];   // new and old exponents
  __shared__ int32_t m_tok[kMembers], m_slot[kMembers];   // a batch: entry, slot, led page, overwritten later
  __shared__ uint8_t m_lead[kMembers], m_dead[kMembers];
  __shared__ int32_t s_range[2], s_wave[4];               // members beyond the chunk: first, last entry; compaction
  __shared__ int32_t s_count, s_grown, s_extra, s_any;
  __shared__ int32_t x_tok[kChunk], x_slot[kChunk], x_lead[kChunk], x_pos[kChunk];   // members beyond the chunk, in no order

  const int tid = threadIdx.x, grp = tid >> 4, u = tid & 15, lane = tid & 63, wave = tid >> 6;
  constexpr int chunk = kChunk / PER, per = PER;       // entries, and 16-lane groups of one
  const int c0 = blockIdx.x * chunk, cn = min(chunk, a.n - c0);
  const T* cos_t = reinterpret_cast<const T*>(a.cos_t);
  const T* sin_t = reinterpret_cast<const T*>(a.sin_t);
  const bool rope = cos_t != nullptr;

  auto valid = [&](int i) {
    const int p = a.page_idx[i], s = a.slot[i];
    bool ok = p >= 0 && p < a.num_pages && s >= 0 && s < a.page_size;
    if (rope) ok = ok && a.positions[i] >= 0 && a.positions[i] < a.max_pos;
    return ok;
  };
  auto tables = [&](int64_t p, float (&c)[2 * E], float (&s)[2 * E]) {
    load_half<T, E>(cos_t + p * D + u * E, c, 0);
    load_half<T, E>(cos_t + p * D + D / 2 + u * E, c, E);
    load_half<T, E>(sin_t + p * D + u * E, s, 0);
    load_half<T, E>(sin_t + p * D + D / 2 + u * E, s, E);
  };

  // ---- everything that depends on no other load leaves first: a 16-lane group's entry
  // (chunk 16: an entry a group; 4: four groups share one's q heads, and its K and V), its
  // K and V rows of the first heads, its first q rows, and the page ids of the scan
  const int h0 = blockIdx.y * a.hkv_share, h1 = min(a.hkv, h0 + a.hkv_share);
  const int own = grp / per, sub = grp % per;
  const bool mine = own < cn;
  const int64_t tok = c0 + min(own, cn - 1);
  const int e_page = a.page_idx[tok], e_slot = a.slot[tok];
  const int64_t e_pos = rope ? a.positions[tok] : 0;
  constexpr int HB = 8 / E;                            // KV heads of a pass (16 values of a row's 16 lanes each, K and V)
  Pack<T, E> k_lo[HB], k_hi[HB], v_lo[HB], v_hi[HB];
  auto load_kv = [&](int h) {
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      if (h + b >= h1) continue;
      if (per == 1 || sub == 0) {
        const T* k = reinterpret_cast<const T*>(a.k) + tok * a.k_sn + (int64_t)(h + b) * a.k_sh + u * E;
        k_lo[b] = *reinterpret_cast<const Pack<T, E>*>(k);
        k_hi[b] = *reinterpret_cast<const Pack<T, E>*>(k + D / 2);
      }
      if (per == 1 || sub == 1) {
        const T* v = reinterpret_cast<const T*>(a.v) + tok * a.v_sn + (int64_t)(h + b) * a.v_sh + u * E;
        v_lo[b] = *reinterpret_cast<const Pack<T, E>*>(v);
        v_hi[b] = *reinterpret_cast<const Pack<T, E>*>(v + D / 2);
      }
    }
  };
  load_kv(h0);
  const int q0 = blockIdx.y * a.hq_share, q1 = min(a.hq, q0 + a.hq_share);
  constexpr int QB = 16 / E;                           // q heads of a pass
  Pack<T, E> q_lo[QB], q_hi[QB];
  auto load_q = [&](int h) {
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      if (h + b * per >= q1) continue;
      const T* src = reinterpret_cast<const T*>(a.q) + tok * a.q_sn + (int64_t)(h + b * per) * D + u * E;
      q_lo[b] = *reinterpret_cast<const Pack<T, E>*>(src);
      q_hi[b] = *reinterpret_cast<const Pack<T, E>*>(src + D / 2);
    }
  };
  load_q(q0 + sub);                                    // (hq is 0 without a rotation)
  constexpr int U = PER == 1 ? 8 : 1;                  // ids of a thread in flight (1: all of kFew entries)
  int ids[U];
  auto load_ids = [&](int j0) {
#pragma unroll
    for (int i = 0; i < U; ++i) ids[i] = j0 + 256 * i + tid < a.n ? a.page_idx[j0 + 256 * i + tid] : -1;
  };
  load_ids(0);

  // ---- the chunk's entries, the tables of a group's
  const bool pos_ok = !rope || (e_pos >= 0 && e_pos < a.max_pos);
  float ct[2 * E], st[2 * E];
  if (rope && pos_ok) tables(e_pos, ct, st);
  if (sub == 0 && u == 0) {
    const bool ok = mine && pos_ok && e_page >= 0 && e_page < a.num_pages && e_slot >= 0 && e_slot < a.page_size;
    s_page[own] = ok ? e_page : -1;
    s_slot[own] = e_slot;
    if (mine && !ok && a.err && blockIdx.y == 0) atomicAdd(a.err, 1);
  }
  if (tid < kChunk) {
    if (tid >= chunk) s_page[tid] = -1;
    s_first[tid] = a.page_size;
  }
  if (tid < 2) s_range[tid] = tid == 0 ? a.n : -1;
  if (tid == 0) s_extra = s_any = 0;
  if (tid < kHeads * kChunk * 2) (&s_amax[0][0][0])[tid] = 0;
  __syncthreads();
  // which entry of the chunk leads its page, which is written again by a later one of the
  // chunk (lane i: entry i; every wave for itself); a 64-bit filter of the pages
  const int w_page = s_page[lane & 15], w_slot = s_slot[lane & 15];
  int w_lead = -1;
  bool w_dead = false;
  uint32_t f0 = 0, f1 = 0;
#pragma unroll
  for (int i = kChunk - 1; i >= 0; --i) {
    const int p = __builtin_amdgcn_readlane(w_page, i), t = __builtin_amdgcn_readlane(w_slot, i);
    if (p < 0) continue;
    if (p == w_page) {
      w_dead = w_dead || (i > (lane & 15) && t == w_slot);
      w_lead = i;
    }
    if (p & 32) f1 |= 1u << (p & 31);
    else f0 |= 1u << (p & 31);
  }
  if (tid < kChunk) {
    s_lead[tid] = w_lead;
    s_dead[tid] = w_dead;
  }
  // up to four led pages (prompts): looked for themselves, not by the filter
  uint32_t leads = (uint32_t)__ballot(lane < kChunk && w_lead == lane);
  const bool few = __builtin_popcount(leads) <= kFewPages, more = few && __builtin_popcount(leads) > 2;
  int f_page[kFewPages], f_lead[kFewPages];
#pragma unroll
  for (int i = 0; i < kFewPages; ++i) {
    f_lead[i] = leads ? __builtin_ctz(leads) : i > 0 ? f_lead[0] : 0;
    f_page[i] = leads ? __builtin_amdgcn_readlane(w_page, f_lead[i]) : i > 0 ? f_page[0] : -1;   // (-1: no page at all)
    leads &= leads - 1;
  }
  __syncthreads();

  // ---- entries of the led pages outside the chunk
  auto lead_of = [&](int p) {
    for (int i = 0; i < cn; ++i)
      if (s_page[i] == p) return s_lead[i];
    return -1;
  };
  auto maybe = [&](int p) { return ((p & 32 ? f1 : f0) >> (p & 31)) & 1u; };
  for (int j0 = 0; j0 < a.n; j0 += 256 * U) {
    uint32_t hits = 0;
    if (few) {
#pragma unroll
      for (int i = 0; i < U; ++i) hits |= ((uint32_t)(ids[i] == f_page[0]) | (uint32_t)(ids[i] == f_page[1])) << i;
      if (more) {
#pragma unroll
        for (int i = 0; i < U; ++i) hits |= ((uint32_t)(ids[i] == f_page[2]) | (uint32_t)(ids[i] == f_page[3])) << i;
      }
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) hits |= maybe(ids[i]) << i;
    }
    if (PER == 1) load_ids(j0 + 256 * U);              // the next ones', ahead of these ones' hits
    while (hits) {
      const int j = j0 + 256 * __builtin_ctz(hits) + tid;
      hits &= hits - 1;
      if (j >= a.n || (j >= c0 && j < c0 + cn)) continue;
      const int p = a.page_idx[j], sl = a.slot[j];       // (one round trip)
      const int64_t at = rope ? a.positions[j] : 0;
      int l = -1;
      if (few) {
#pragma unroll
        for (int f = 0; f < kFewPages; ++f) l = p == f_page[f] ? f_lead[f] : l;
      } else if (p >= 0) {
        l = lead_of(p);
      }
      if (p < 0 || l < 0 || sl < 0 || sl >= a.page_size || (rope && (at < 0 || at >= a.max_pos))) continue;
      if (j < c0) {
        s_first[l] = -1;                               // led by an earlier workgroup
      } else {
        atomicMin(&s_range[0], j);
        atomicMax(&s_range[1], j);
        const int x = atomicAdd(&s_extra, 1);
        if (x < kChunk) {
          x_tok[x] = j;
          x_slot[x] = sl;
          x_lead[x] = l;
          x_pos[x] = (int32_t)at;
        }
      }
    }
  }

  // ---- q rows
  if (mine && pos_ok) {
    T* dst = reinterpret_cast<T*>(a.q_out) + tok * a.hq * D + u * E;
    for (int h = q0 + sub; h < q1; h += QB * per) {
      Pack<T, E> lo[QB], hi[QB];
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        lo[b] = q_lo[b];
        hi[b] = q_hi[b];
      }
      load_q(h + QB * per);                            // the next pass's, ahead of this one's products
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        if (h + b * per >= q1) continue;
        float x[2 * E];
        unpack<T, E>(lo[b], x, 0);
        unpack<T, E>(hi[b], x, E);
        rotate<E>(x, ct, st);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          lo[b].x[e] = from_f32<T>(x[e]);
          hi[b].x[e] = from_f32<T>(x[E + e]);
        }
        *reinterpret_cast<Pack<T, E>*>(dst + (h + b * per) * D) = lo[b];
        *reinterpret_cast<Pack<T, E>*>(dst + (h + b * per) * D + D / 2) = hi[b];
      }
    }
  }

  if (h0 >= h1) return;
  __syncthreads();

  // ---- batches of members: the chunk's own, then the later entries in tiles.  One
  // tile's members join the chunk's; more tiles are batches of their own, gone through
  // once for the largest values and once more to write.
  const int jb = s_range[0], je = s_range[1] + 1;     // later members lie in [jb, je)
  const int tiles = je > jb ? (je - jb + kTile - 1) / kTile : 0;
  int members = 0;
  // batch 0: the chunk's own and (a single tile) the tile's; batch b > 0: tile b - 1
  auto collect = [&](int b) {
    __syncthreads();
    if (b == 0) {
      if (wave == 0) {
        const bool led = lane < cn && s_lead[min(lane, kChunk - 1)] >= 0 && s_first[s_lead[min(lane, kChunk - 1)]] >= 0;
        const uint64_t bal = __ballot(led);
        if (led) {
          const int at = __popcll(bal & ((1ull << lane) - 1));
          m_tok[at] = c0 + lane;
          m_slot[at] = s_slot[lane];
          m_lead[at] = (uint8_t)s_lead[lane];
        }
        if (lane == 0) s_count = __popcll(bal);
      }
      __syncthreads();
      members = s_count;
    } else {
      members = 0;
    }
    if (tiles > 0 && (b > 0 || tiles == 1)) {
      const int j = jb + (b > 0 ? b - 1 : 0) * kTile + tid;
      int l = -1;
      if (j < je) {
        const int p = a.page_idx[j];
        if (p >= 0 && maybe(p) && valid(j)) {
          l = lead_of(p);
          if (l >= 0 && s_first[l] < 0) l = -1;
        }
      }
      const uint64_t bal = __ballot(l >= 0);
      if (lane == 0) s_wave[wave] = __popcll(bal);
      __syncthreads();
      int at = members + __popcll(bal & ((1ull << lane) - 1));
      for (int w = 0; w < wave; ++w) at += s_wave[w];
      if (l >= 0) {
        m_tok[at] = j;
        m_slot[at] = a.slot[j];
        m_lead[at] = (uint8_t)l;
      }
      members += s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
    }
    __syncthreads();
    // an entry whose (page, slot) a later one of the batch names again is not written
    for (int m = tid; m < members; m += 256) {
      bool dead = false;
      for (int o = m + 1; o < members; ++o) dead = dead || (m_slot[o] == m_slot[m] && m_lead[o] == m_lead[m]);
      m_dead[m] = dead;
    }
    __syncthreads();
  };
  // a member's K (sel 0) or V row of a head
  auto row = [&](int tok, int sel, int h, float (&x)[2 * E]) {
    const T* src = reinterpret_cast<const T*>(sel ? a.v : a.k) + (int64_t)tok * (sel ? a.v_sn : a.k_sn) +
                   (int64_t)h * (sel ? a.v_sh : a.k_sh) + u * E;
    load_half<T, E>(src, x, 0);
    load_half<T, E>(src + D / 2, x, E);
    if (!sel && rope) {
      float c[2 * E], s[2 * E];
      tables(a.positions[tok], c, s);
      rotate<E>(x, c, s);
    }
  };
  auto take_max = [&](int lead, int sel, int hi, const float (&x)[2 * E]) {
    float mx = 0.f;
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) {
      const float y = fabsf(x[e]);
      mx = fmaxf(mx, y < INFINITY ? y : 0.f);
    }
    mx = fminf(mx, largest<T>());
    mx = max16(mx);
    if (u == 0) atomicMax(&s_amax[hi][lead][sel], __float_as_uint(mx));
  };
  auto store = [&](int l, int slot, int sel, int h, int hi, const float (&x)[2 * E]) {
    const float inv = exp2i(-s_exp[hi][l][sel]), top = largest<T>();
    float y[2 * E];
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) {
      // (an infinity stays one, and becomes a NaN code)
      const float z = fabsf(x[e]) < INFINITY ? fminf(fmaxf(x[e], -top), top) : x[e];
      y[e] = z * inv;
    }
    uint8_t* dst = a.kv + ((((int64_t)s_page[l] * 2 + sel) * a.page_size + slot) * a.hkv + h) * D + u * E;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int o = half * E;
      uint8_t* d = dst + half * (D / 2);
      if constexpr (E == 2) {
        *reinterpret_cast<uint16_t*>(d) = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[o], y[o + 1], 0, false);
      } else if constexpr (E == 4) {
        *reinterpret_cast<uint32_t*>(d) = codes4(y[o], y[o + 1], y[o + 2], y[o + 3]);
      } else {
        const uint2 w = {codes4(y[o], y[o + 1], y[o + 2], y[o + 3]), codes4(y[o + 4], y[o + 5], y[o + 6], y[o + 7])};
        *reinterpret_cast<uint2*>(d) = w;
      }
    }
  };

  // the old exponents of a pass's blocks, ahead of what they are compared with: thread
  // (head, page, K / V)
  auto scale_at = [&](int h) { return a.scale + ((int64_t)s_page[(tid >> 1) & 15] * 2 + (tid & 1)) * a.hkv + h; };
  auto is_block = [&](int l) { return s_lead[l] == l && s_first[l] >= 0 && s_first[l] < a.page_size; };
  auto old_exp = [&](int h, int nh) {
    const int l = (tid >> 1) & 15, hi = tid >> 5;
    return hi < nh && is_block(l) && s_first[l] > 0 ? min((int)*scale_at(h + hi) - 127, 120) : 0;   // (120: a bf16 block's most)
  };
  auto new_exp = [&](int h, int nh, int old) {
    const int l = (tid >> 1) & 15, sel = tid & 1, hi = tid >> 5;
    if (hi >= nh) return;
    int e = 0;
    if (is_block(l)) {
      e = block_exp(s_amax[hi][l][sel]);
      if (s_first[l] > 0) {
        e = max(e, old);
        if (e > old) s_grown = 1;
      } else {
        old = e;
      }
      *scale_at(h + hi) = (uint8_t)(e + 127);
    } else {
      old = 0;
    }
    s_exp[hi][l][sel] = e;
    s_old[hi][l][sel] = old;
    s_amax[hi][l][sel] = 0;
  };
  // tokens written before, where a scale grew
  auto rescale = [&](int h, int nh) {
    for (int hi = 0; hi < nh; ++hi)
      for (int l = 0; l < cn; ++l)
        for (int sel = 0; sel < 2; ++sel) {
          const int by = s_old[hi][l][sel] - s_exp[hi][l][sel];
          if (by >= 0) continue;
          const float f = exp2i(max(by, -126));
          for (int t = grp; t < s_first[l]; t += 16) {
            uint8_t* d = a.kv + ((((int64_t)s_page[l] * 2 + sel) * a.page_size + t) * a.hkv + h + hi) * D + u * (D / 16);
#pragma unroll
            for (int w = 0; w < D / 64; ++w) {
              typedef float f2 __attribute__((ext_vector_type(2)));
              const int c = *reinterpret_cast<const int*>(d + 4 * w);
              const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi2 = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
              *reinterpret_cast<uint32_t*>(d + 4 * w) = codes4(lo.x * f, lo.y * f, hi2.x * f, hi2.y * f);
            }
          }
        }
  };

  // ---- at most 16 entries outside the chunk belong to its pages (decode steps, prompts on
  // pages of up to 16 tokens): the groups' own rows, which are there already, and one
  // such entry a group
  const int extra = __builtin_amdgcn_readfirstlane(s_extra);
  if (extra <= kChunk) {
    const int l = s_lead[own], xl = grp < extra ? x_lead[grp] : -1;
    const bool led = mine && l >= 0 && s_first[max(l, 0)] >= 0, xled = xl >= 0 && s_first[max(xl, 0)] >= 0;
    const int xs = xl >= 0 ? x_slot[grp] : 0, xt = xl >= 0 ? x_tok[grp] : 0;
    if (led || xled) s_any = 1;
    __syncthreads();
    if (!s_any) return;
    Pack<T, E> xk_lo[HB], xk_hi[HB], xv_lo[HB], xv_hi[HB];
    auto load_x = [&](int h) {
#pragma unroll
      for (int b = 0; b < HB; ++b) {
        if (!xled || h + b >= h1) continue;
        const T* k = reinterpret_cast<const T*>(a.k) + (int64_t)xt * a.k_sn + (int64_t)(h + b) * a.k_sh + u * E;
        const T* v = reinterpret_cast<const T*>(a.v) + (int64_t)xt * a.v_sn + (int64_t)(h + b) * a.v_sh + u * E;
        xk_lo[b] = *reinterpret_cast<const Pack<T, E>*>(k);
        xk_hi[b] = *reinterpret_cast<const Pack<T, E>*>(k + D / 2);
        xv_lo[b] = *reinterpret_cast<const Pack<T, E>*>(v);
        xv_hi[b] = *reinterpret_cast<const Pack<T, E>*>(v + D / 2);
      }
    };
    if (extra > 0) load_x(h0);
    float xc[2 * E], xn[2 * E];
    if (rope && xled) tables(x_pos[grp], xc, xn);
    if (u == 0) {
      if (led && sub == 0) atomicMin(&s_first[l], e_slot);
      if (xled) atomicMin(&s_first[xl], xs);
    }
    // (of entries with the same page and slot the last is written)
    bool write = led && !s_dead[own], xwrite = xled;
    for (int o = 0; o < extra; ++o) {
      const int ol = x_lead[o], os = x_slot[o];
      write = write && !(ol == l && os == e_slot);
      xwrite = xwrite && !(ol == xl && os == xs && x_tok[o] > xt);
    }
    __syncthreads();
    for (int h = h0; h < h1; h += HB) {
      const int nh = min(HB, h1 - h), old = old_exp(h, nh);
      if (h > h0) {
        load_kv(h);
        if (extra > 0) load_x(h);
      }
      float xk[HB][2 * E], xv[HB][2 * E];
#pragma unroll
      for (int b = 0; b < HB; ++b) {
        if (!led || b >= nh) continue;
        if (per == 1 || sub == 0) {
          unpack<T, E>(k_lo[b], xk[b], 0);
          unpack<T, E>(k_hi[b], xk[b], E);
          if (rope) rotate<E>(xk[b], ct, st);
          take_max(l, 0, b, xk[b]);
        }
        if (per == 1 || sub == 1) {
          unpack<T, E>(v_lo[b], xv[b], 0);
          unpack<T, E>(v_hi[b], xv[b], E);
          take_max(l, 1, b, xv[b]);
        }
      }
      auto x_row = [&](int sel, int b, float (&x)[2 * E]) {
        unpack<T, E>(sel ? xv_lo[b] : xk_lo[b], x, 0);
        unpack<T, E>(sel ? xv_hi[b] : xk_hi[b], x, E);
        if (!sel && rope) rotate<E>(x, xc, xn);
      };
      if (extra > 0) {
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          if (!xled || b >= nh) continue;
#pragma unroll
          for (int sel = 0; sel < 2; ++sel) {
            float x[2 * E];
            x_row(sel, b, x);
            take_max(xl, sel, b, x);
          }
        }
      }
      if (tid == 0) s_grown = 0;
      __syncthreads();
      new_exp(h, nh, old);
      __syncthreads();
#pragma unroll
      for (int b = 0; b < HB; ++b) {
        if (!write || b >= nh) continue;
        if (per == 1 || sub == 0) store(l, e_slot, 0, h + b, b, xk[b]);
        if (per == 1 || sub == 1) store(l, e_slot, 1, h + b, b, xv[b]);
      }
      if (extra > 0) {
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          if (!xwrite || b >= nh) continue;
#pragma unroll
          for (int sel = 0; sel < 2; ++sel) {
            float x[2 * E];
            x_row(sel, b, x);
            store(xl, xs, sel, h + b, b, x);
          }
        }
      }
      if (s_grown) rescale(h, nh);
      __syncthreads();
    }
    return;
  }

  collect(0);
  const bool single = tiles <= 1;
  if (single && members == 0) return;
  for (int m = tid; m < members; m += 256) atomicMin(&s_first[m_lead[m]], m_slot[m]);
  for (int b = 1; !single && b <= tiles; ++b) {
    collect(b);
    for (int m = tid; m < members; m += 256) atomicMin(&s_first[m_lead[m]], m_slot[m]);
  }
  __syncthreads();                                   // the least slots are known
  // a few members: a head's rows in registers, one or two a group
  auto held = [&](auto mp_) {
    constexpr int MP = decltype(mp_)::value;
    float c[MP][2 * E], s[MP][2 * E];
#pragma unroll
    for (int m = 0; m < MP; ++m)
      if (rope && grp + 16 * m < members) tables(a.positions[m_tok[grp + 16 * m]], c[m], s[m]);
    for (int h = h0; h < h1; ++h) {
      const int old = old_exp(h, 1);
      float x[MP][2][2 * E];
#pragma unroll
      for (int m = 0; m < MP; ++m) {
        if (grp + 16 * m >= members) continue;
        const int64_t t = m_tok[grp + 16 * m];
        const T* k = reinterpret_cast<const T*>(a.k) + t * a.k_sn + (int64_t)h * a.k_sh + u * E;
        const T* v = reinterpret_cast<const T*>(a.v) + t * a.v_sn + (int64_t)h * a.v_sh + u * E;
        load_half<T, E>(k, x[m][0], 0);
        load_half<T, E>(k + D / 2, x[m][0], E);
        load_half<T, E>(v, x[m][1], 0);
        load_half<T, E>(v + D / 2, x[m][1], E);
      }
#pragma unroll
      for (int m = 0; m < MP; ++m) {
        if (grp + 16 * m >= members) continue;
        if (rope) rotate<E>(x[m][0], c[m], s[m]);
        take_max(m_lead[grp + 16 * m], 0, 0, x[m][0]);
        take_max(m_lead[grp + 16 * m], 1, 0, x[m][1]);
      }
      if (tid == 0) s_grown = 0;
      __syncthreads();
      new_exp(h, 1, old);
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MP; ++m) {
        const int i = grp + 16 * m;
        if (i >= members || m_dead[i]) continue;
        store(m_lead[i], m_slot[i], 0, h, 0, x[m][0]);
        store(m_lead[i], m_slot[i], 1, h, 0, x[m][1]);
      }
      if (s_grown) rescale(h, 1);
      __syncthreads();
    }
  };
  if (single && members <= 32) {
    held(std::integral_constant<int, 2>());
  } else {
    for (int h = h0; h < h1; ++h) {
      const int old = old_exp(h, 1);
      for (int b = 0; b <= (single ? 0 : tiles); ++b) {
        if (!single) collect(b);
        for (int r = grp; r < 2 * members; r += 16) {
          float x[2 * E];
          row(m_tok[r >> 1], r & 1, h, x);
          take_max(m_lead[r >> 1], r & 1, 0, x);
        }
      }
      if (tid == 0) s_grown = 0;
      __syncthreads();
      new_exp(h, 1, old);
      __syncthreads();
      for (int b = 0; b <= (single ? 0 : tiles); ++b) {
        if (!single) collect(b);
        for (int r = grp; r < 2 * members; r += 16) {
          const int m = r >> 1;
          if (m_dead[m]) continue;
          float x[2 * E];
          row(m_tok[m], r & 1, h, x);
          store(m_lead[m], m_slot[m], r & 1, h, 0, x);
        }
      }
      if (s_grown) rescale(h, 1);
      __syncthreads();
    }
  }
}

// grid.x = copy entry, grid.y = layer * 2 + K / V: the first len tokens' codes and,
// for any token at all, the page's scales of the source.  (40 pages of 16 tokens on 8
// layers: 4.9 us, a launch and two round trips.)
__global__ __launch_bounds__(256) void copy_kernel(uint8_t* pool, int64_t layer_stride, uint8_t* scales, int64_t scale_stride,
                                                  int num_pages, int page_size, int hkv, int d, const int32_t* src,
                                                  const int32_t* dst, const int32_t* len, const int32_t* count, int32_t* err) {
  const int c = blockIdx.x;
  if (count && c >= *count) return;
  const int layer = blockIdx.y >> 1, sel = blockIdx.y & 1;
  const int s = src[c], t = dst[c], l = len[c];
  if (s < 0 || s >= num_pages || t < 0 || t >= num_pages || l < 0 || l > page_size) {
    if (err && threadIdx.x == 0 && blockIdx.y == 0) atomicAdd(err, 1);
    return;
  }
  if (l == 0) return;
  const int64_t plane = (int64_t)page_size * hkv * d, chunks = (int64_t)l * hkv * d / 16;
  const uint4* sp = reinterpret_cast<const uint4*>(pool + layer * layer_stride + ((int64_t)s * 2 + sel) * plane);
  uint4* dp = reinterpret_cast<uint4*>(pool + layer * layer_stride + ((int64_t)t * 2 + sel) * plane);
  for (int64_t i = threadIdx.x; i < chunks; i += 256) dp[i] = sp[i];
  const uint8_t* ss = scales + layer * scale_stride + ((int64_t)s * 2 + sel) * hkv;
  uint8_t* ds = scales + layer * scale_stride + ((int64_t)t * 2 + sel) * hkv;
  for (int h = threadIdx.x; h < hkv; h += 256) ds[h] = ss[h];
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ uint32_t value2(uint32_t codes, float scale, bool high);
template <>
__device__ __forceinline__ uint32_t value2<bf16_t>(uint32_t codes, float scale, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)codes, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)codes, scale, false));
}
template <>
__device__ __forceinline__ uint32_t value2<f16_t>(uint32_t codes, float scale, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)codes, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)codes, scale, false));
}

// Values of `planes` (page, K / V) planes, 16 codes a thread; `step` 2 takes the K or
// the V planes only (from plane `first`).  Bound by the bytes, 1 read and 2 written a value:
// 168 pages of 16 tokens on 8 layers (8 heads of 128, 132 MB) in 21 us, some of it from cache.
template <typename T>
__global__ __launch_bounds__(256) void values_kernel(const uint8_t* kv, const uint8_t* scale, T* out, int64_t planes,
                                                    int page_size, int hkv, int d, int first, int step) {
  const int per_row = d / 16;
  const int64_t per = (int64_t)page_size * hkv * per_row, total = planes * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t pl = i / per;
    const int in = (int)(i - pl * per), h = (in / per_row) % hkv;
    const int64_t from = first + pl * step;
    const float s = __uint_as_float((uint32_t)scale[from * hkv + h] << 23);
    const u32x4 c = *reinterpret_cast<const u32x4*>(kv + (from * per + in) * 16);
    u32x4 o[2];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      o[w >> 1][2 * (w & 1)] = value2<T>(c[w], s, false);
      o[w >> 1][2 * (w & 1) + 1] = value2<T>(c[w], s, true);
    }
    u32x4* to = reinterpret_cast<u32x4*>(out + i * 16);
    to[0] = o[0];
    to[1] = o[1];
  }
}

static int check_cache(const void* kv, const void* scale, int num_pages, int page_size, int hkv, int d) {
  BE_REQUIRE(kv && scale, "null pointer");
  BE_REQUIRE(num_pages > 0 && page_size > 0 && hkv > 0, "bad cache shape");
  if (d != 64 && d != 128 && d != 256) return fail(BE_ERR_UNSUPPORTED, "8-bit cache: head_dim %d, kernels exist for 64, 128, 256", d);
  BE_REQUIRE((reinterpret_cast<uintptr_t>(kv) & 15) == 0, "the 8-bit cache must be 16-byte aligned");
  return BE_OK;
}

// Few entries (a decode step): four a workgroup and one KV head each, so that their rows
// spread over the CUs; many: 16 (a page's worth), and as few shares of the heads as leave
// every CU four workgroups.  At 32 heads of 128 over 8, four / 16 a workgroup: 128 lone
// tokens 9.0 / 12.2 us, 256 9.9 / 12.8, 512 15.5 / 15.2; prompts of 256 tokens 13.3 / 10.3,
// of 512 22.1 / 11.2.
template <typename T, int D>
static void launch_per(const AppendArgs& a, dim3 grid, hipStream_t st) {
  if (a.n <= kFew) append_kernel<T, D, 4><<<grid, 256, 0, st>>>(a);
  else append_kernel<T, D, 1><<<grid, 256, 0, st>>>(a);
}
static int launch_append(AppendArgs& a, int dtype, int d, hipStream_t st) {
  const int chunk = a.n <= kFew ? kChunk / 4 : kChunk;
  const unsigned gx = (unsigned)((a.n + chunk - 1) / chunk);
  const int shares = (int)std::min<int64_t>(a.hkv, std::max<int64_t>(1, (1024 + gx - 1) / gx));
  a.hkv_share = (a.hkv + shares - 1) / shares;
  a.hq_share = (a.hq + shares - 1) / shares;
  const dim3 grid(gx, (unsigned)shares);
#define BE_APPEND(TY)                                       \
  switch (d) {                                              \
    case 64: launch_per<TY, 64>(a, grid, st); break;        \
    case 128: launch_per<TY, 128>(a, grid, st); break;      \
    default: launch_per<TY, 256>(a, grid, st); break;       \
  }
  if (dtype == BE_BF16) { BE_APPEND(bf16_t) } else { BE_APPEND(f16_t) }
#undef BE_APPEND
  BE_HIP_CHECK(hipGetLastError());
  return BE_OK;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace kv8
}  // namespace be

extern "C" {

int be_kv8_append(void* kv_layer, void* scale_layer, int dtype, int num_pages, int page_size, int num_kv_heads, int head_dim,
                  const int32_t* page_idx, const int32_t* pos, const void* k, int64_t k_stride_n, int64_t k_stride_h,
                  const void* v, int64_t v_stride_n, int64_t v_stride_h, int n, int32_t* err_count, void* stream) {
  using namespace be;
  BE_REQUIRE(n >= 0, "n must be >= 0");
  if (n == 0) return BE_OK;
  BE_REQUIRE(page_idx && pos && k && v, "null pointer");
  BE_REQUIRE(dtype == BE_F16 || dtype == BE_BF16, "an 8-bit cache takes fp16 / bf16 rows");
  if (const int rc = kv8::check_cache(kv_layer, scale_layer, num_pages, page_size, num_kv_heads, head_dim)) return rc;
  BE_REQUIRE(kv8::aligned16(k) && kv8::aligned16(v) && ((k_stride_n | k_stride_h | v_stride_n | v_stride_h) & 7) == 0,
             "rows of k and v must start on 16 bytes");
  kv8::AppendArgs a{};
  a.k = k; a.v = v;
  a.k_sn = k_stride_n; a.k_sh = k_stride_h; a.v_sn = v_stride_n; a.v_sh = v_stride_h;
  a.kv = static_cast<uint8_t*>(kv_layer); a.scale = static_cast<uint8_t*>(scale_layer);
  a.page_idx = page_idx; a.slot = pos; a.err = err_count;
  a.n = n; a.hkv = num_kv_heads; a.num_pages = num_pages; a.page_size = page_size;
  return kv8::launch_append(a, dtype, head_dim, reinterpret_cast<hipStream_t>(stream));
}

int be_kv8_rope_append(const void* qkv, int64_t qkv_stride_n, int dtype, int n, int num_qo_heads, int num_kv_heads,
                       int head_dim, const int64_t* positions, const void* cos_table, const void* sin_table,
                       int max_position, void* q_out, void* kv_layer, void* scale_layer, int num_pages, int page_size,
                       const int32_t* page_idx, const int32_t* slot, int32_t* err_count, void* stream) {
  using namespace be;
  BE_REQUIRE(n >= 0, "n must be >= 0");
  if (n == 0) return BE_OK;
  BE_REQUIRE(qkv && positions && cos_table && sin_table && q_out && page_idx && slot, "null pointer");
  BE_REQUIRE(dtype == BE_F16 || dtype == BE_BF16, "an 8-bit cache takes fp16 / bf16 rows");
  BE_REQUIRE(num_qo_heads > 0 && num_kv_heads > 0 && max_position > 0, "bad head or table shape");
  if (const int rc = kv8::check_cache(kv_layer, scale_layer, num_pages, page_size, num_kv_heads, head_dim)) return rc;
  BE_REQUIRE(qkv_stride_n >= (int64_t)(num_qo_heads + 2 * num_kv_heads) * head_dim, "qkv row stride too small");
  BE_REQUIRE(kv8::aligned16(qkv) && (qkv_stride_n & 7) == 0 && kv8::aligned16(cos_table) && kv8::aligned16(sin_table) &&
                 kv8::aligned16(q_out),
             "rows of qkv, the tables and q_out must start on 16 bytes");
  const char* row = static_cast<const char*>(qkv);
  kv8::AppendArgs a{};
  a.q = qkv;
  a.k = row + (int64_t)num_qo_heads * head_dim * 2;
  a.v = row + (int64_t)(num_qo_heads + num_kv_heads) * head_dim * 2;
  a.q_sn = a.k_sn = a.v_sn = qkv_stride_n;
  a.k_sh = a.v_sh = head_dim;
  a.cos_t = cos_table; a.sin_t = sin_table; a.positions = positions; a.q_out = q_out;
  a.kv = static_cast<uint8_t*>(kv_layer); a.scale = static_cast<uint8_t*>(scale_layer);
  a.page_idx = page_idx; a.slot = slot; a.err = err_count;
  a.n = n; a.hq = num_qo_heads; a.hkv = num_kv_heads; a.num_pages = num_pages; a.page_size = page_size;
  a.max_pos = max_position;
  return kv8::launch_append(a, dtype, head_dim, reinterpret_cast<hipStream_t>(stream));
}

int be_kv8_page_copy(void* kv_pool, int64_t layer_stride_bytes, void* scale_pool, int64_t scale_stride_bytes, int num_layers,
                     int num_pages, int page_size, int num_kv_heads, int head_dim, const int32_t* src, const int32_t* dst,
                     const int32_t* len, const int32_t* count, int n, int32_t* err_count, void* stream) {
  using namespace be;
  BE_REQUIRE(n >= 0 && num_layers >= 0, "negative count");
  if (n == 0 || num_layers == 0) return BE_OK;
  BE_REQUIRE(src && dst && len, "null pointer");
  if (const int rc = kv8::check_cache(kv_pool, scale_pool, num_pages, page_size, num_kv_heads, head_dim)) return rc;
  BE_REQUIRE(num_layers == 1 || (layer_stride_bytes >= (int64_t)num_pages * 2 * page_size * num_kv_heads * head_dim &&
                                 layer_stride_bytes % 16 == 0 &&
                                 scale_stride_bytes >= (int64_t)num_pages * 2 * num_kv_heads),
             "layer strides %lld / %lld smaller than one layer, or not 16-byte aligned", (long long)layer_stride_bytes,
             (long long)scale_stride_bytes);
  BE_REQUIRE(num_layers <= 32767, "too many layers");
  kv8::copy_kernel<<<dim3(n, num_layers * 2), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
      static_cast<uint8_t*>(kv_pool), layer_stride_bytes, static_cast<uint8_t*>(scale_pool), scale_stride_bytes, num_pages,
      page_size, num_kv_heads, head_dim, src, dst, len, count, err_count);
  BE_HIP_CHECK(hipGetLastError());
  return BE_OK;
}

int be_kv8_values(const void* kv, const void* scale, int dtype, int num_pages, int page_size, int num_kv_heads, int head_dim,
                  int which, void* out, void* stream) {
  using namespace be;
  BE_REQUIRE(num_pages >= 0 && which >= -1 && which <= 1, "bad page count or plane choice");
  if (num_pages == 0) return BE_OK;
  BE_REQUIRE(dtype == BE_F16 || dtype == BE_BF16, "values of an 8-bit cache are fp16 / bf16");
  if (const int rc = kv8::check_cache(kv, scale, num_pages, page_size, num_kv_heads, head_dim)) return rc;
  BE_REQUIRE(out && kv8::aligned16(out), "out must be 16-byte aligned");
  const int64_t planes = which < 0 ? 2 * (int64_t)num_pages : num_pages;
  const int64_t threads = planes * page_size * num_kv_heads * (head_dim / 16);
  const unsigned blocks = (unsigned)std::min<int64_t>((threads + 255) / 256, 1 << 20);
  const int first = which == 1 ? 1 : 0, step = which < 0 ? 1 : 2;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == BE_BF16)
    kv8::values_kernel<bf16_t><<<blocks, 256, 0, st>>>(static_cast<const uint8_t*>(kv), static_cast<const uint8_t*>(scale),
                                                      static_cast<bf16_t*>(out), planes, page_size, num_kv_heads, head_dim,
                                                      first, step);
  else
    kv8::values_kernel<f16_t><<<blocks, 256, 0, st>>>(static_cast<const uint8_t*>(kv), static_cast<const uint8_t*>(scale),
                                                     static_cast<f16_t*>(out), planes, page_size, num_kv_heads, head_dim,
                                                     first, step);
  BE_HIP_CHECK(hipGetLastError());
  return BE_OK;
}

}  // extern "C"
