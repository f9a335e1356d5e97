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

#include "common.h"

namespace be {
namespace kv8 {

constexpr int kLeastExp = -100;        // (2^126 of its inverse stays finite)
constexpr int kChunk = 16;             // entries of a workgroup, at most
constexpr int kTile = 256;             // entries of a scan step, members of a batch beyond the chunk's
constexpr int kMembers = kChunk + kTile;

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

struct AppendArgs {
  const void *q, *k, *v;               // rows of head_dim elements, 16-byte aligned; q: with cos only
  int64_t q_sn, k_sn, k_sh, v_sn, v_sh;
  const void *cos_t, *sin_t;           // [max_pos, head_dim], null: no rotation and no q
  const int64_t* positions;
  void* q_out;                         // [n, hq, head_dim]
  uint8_t *kv, *scale;
  const int32_t *page_idx, *slot;
  int32_t* err;
  int n, hq, hkv, num_pages, page_size, max_pos, chunk;
};

// One row of a head over 16 lanes: lane u holds elements u E .. + E - 1 of each half,
// E = D / 32, in v[0..E) and v[E..2E).
template <typename T, int E>
__device__ __forceinline__ void load_half(const T* p, float (&v)[2 * E], int at) {
  struct alignas(2 * E) Pack { T x[E]; };
  const Pack pk = *reinterpret_cast<const Pack*>(p);
#pragma unroll
  for (int e = 0; e < E; ++e) v[at + e] = to_f32(pk.x[e]);
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
// What bounds it: a decode step's launch is a chain of round trips (indices, rows,
// tables, the old scale); prompts are bound by the rows' bytes.
template <typename T, int D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int E = D / 32;
  __shared__ int32_t s_page[kChunk], s_lead[kChunk];      // the chunk's pages (-1: not this workgroup's), and which lead
  __shared__ int32_t s_first[kChunk];                     // per led page: least slot written
  __shared__ uint32_t s_amax[2][kChunk][2];               // per led page, K / V: bits of the largest finite |x|
  __shared__ int32_t s_exp[kChunk][2], s_old[kChunk][2];  // new and old exponents
  __shared__ int32_t m_tok[kMembers], m_slot[kMembers];   // a batch: entry, slot, led page, overwritten later
  __shared__ uint8_t m_lead[kMembers], m_dead[kMembers];
  __shared__ int32_t s_range[2], s_wave[4];               // members beyond the chunk: first, last entry; compaction
  __shared__ int32_t s_count, s_grown;

  const int tid = threadIdx.x, grp = tid >> 4, u = tid & 15, lane = tid & 63, wave = tid >> 6;
  const int c0 = blockIdx.x * a.chunk, cn = min(a.chunk, a.n - c0);
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

  // ---- the chunk's entries
  if (tid < kChunk) {
    int p = -1;
    if (tid < cn) {
      if (valid(c0 + tid)) p = a.page_idx[c0 + tid];
      else if (a.err && blockIdx.y == 0) atomicAdd(a.err, 1);
    }
    s_page[tid] = p;
    s_first[tid] = a.page_size;
  }
  if (tid < 2) s_range[tid] = tid == 0 ? a.n : -1;
  if (tid < 2 * kChunk) s_amax[0][tid >> 1][tid & 1] = s_amax[1][tid >> 1][tid & 1] = 0;
  __syncthreads();
  // which entry of the chunk leads its page; a 64-bit filter of the led pages
  uint64_t filter = 0;
  for (int i = 0; i < cn; ++i)
    if (s_page[i] >= 0) filter |= 1ull << (s_page[i] & 63);
  if (tid < kChunk) {
    int lead = -1;
    if (s_page[tid] >= 0) {
      lead = tid;
      for (int i = tid - 1; i >= 0; --i)
        if (s_page[i] == s_page[tid]) lead = i;
    }
    s_lead[tid] = lead;
  }
  __syncthreads();

  // ---- entries of the led pages outside the chunk
  {
    auto look = [&](int j, int p) {
      if ((uint32_t)p >= (uint32_t)a.num_pages || !((filter >> (p & 63)) & 1)) return;
      int l = -1;
      for (int i = 0; i < cn; ++i)
        if (s_page[i] == p) { l = s_lead[i]; break; }
      if (l < 0 || (j >= c0 && j < c0 + cn) || !valid(j)) return;
      if (j < c0) {
        s_first[l] = -1;                             // led by an earlier workgroup
      } else {
        atomicMin(&s_range[0], j);
        atomicMax(&s_range[1], j);
      }
    };
    // (the least slot is taken below: s_first < 0 marks a page that is not led here)
    constexpr int U = 8;
    for (int j0 = tid; j0 < a.n; j0 += 256 * U) {
      int p[U];
#pragma unroll
      for (int i = 0; i < U; ++i) p[i] = j0 + 256 * i < a.n ? a.page_idx[j0 + 256 * i] : -1;
#pragma unroll
      for (int i = 0; i < U; ++i) look(j0 + 256 * i, p[i]);
    }
  }

  // ---- q rows of the chunk
  if (rope && a.hq) {
    const int h0 = (int)((int64_t)a.hq * blockIdx.y / gridDim.y), h1 = (int)((int64_t)a.hq * (blockIdx.y + 1) / gridDim.y);
    const int nh = h1 - h0;
    for (int r = grp; r < cn * nh; r += 16) {
      const int i = c0 + r / nh, h = h0 + r % nh;
      const int64_t p = a.positions[i];
      if (p < 0 || p >= a.max_pos) continue;
      const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)i * a.q_sn + (int64_t)h * D + u * E;
      float x[2 * E], c[2 * E], s[2 * E];
      load_half<T, E>(src, x, 0);
      load_half<T, E>(src + D / 2, x, E);
      tables(p, c, s);
      rotate<E>(x, c, s);
      struct alignas(2 * E) Pack { T x[E]; } lo, hi;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        lo.x[e] = from_f32<T>(x[e]);
        hi.x[e] = from_f32<T>(x[E + e]);
      }
      T* dst = reinterpret_cast<T*>(a.q_out) + ((int64_t)i * a.hq + h) * D + u * E;
      *reinterpret_cast<Pack*>(dst) = lo;
      *reinterpret_cast<Pack*>(dst + D / 2) = hi;
    }
  }

  const int h0 = (int)((int64_t)a.hkv * blockIdx.y / gridDim.y), h1 = (int)((int64_t)a.hkv * (blockIdx.y + 1) / gridDim.y);
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
        const bool mine = lane < cn && s_lead[min(lane, kChunk - 1)] >= 0 && s_first[s_lead[min(lane, kChunk - 1)]] >= 0;
        const uint64_t bal = __ballot(mine);
        if (mine) {
          const int at = __popcll(bal & ((1ull << lane) - 1));
          m_tok[at] = c0 + lane;
          m_slot[at] = a.slot[c0 + lane];
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
        if ((uint32_t)p < (uint32_t)a.num_pages && ((filter >> (p & 63)) & 1) && valid(j)) {
          for (int i = 0; i < cn; ++i)
            if (s_page[i] == p) { l = s_lead[i]; break; }
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
  auto take_max = [&](int m, int sel, int buf, const float (&x)[2 * E]) {
    float mx = 0.f;
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) {
      const float y = fabsf(x[e]);
      mx = fmaxf(mx, y < INFINITY ? y : 0.f);
    }
    mx = fminf(mx, largest<T>());
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 16));
    if (u == 0) atomicMax(&s_amax[buf][m_lead[m]][sel], __float_as_uint(mx));
  };
  auto store = [&](int m, int sel, int h, const float (&x)[2 * E]) {
    if (m_dead[m]) return;
    const int l = m_lead[m];
    const float inv = exp2i(-s_exp[l][sel]), top = largest<T>();
    float y[2 * E];
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) {
      // (an infinity stays one, and becomes a NaN code)
      const float z = fabsf(x[e]) < INFINITY ? fminf(fmaxf(x[e], -top), top) : x[e];
      y[e] = z * inv;
    }
    uint8_t* dst = a.kv + ((((int64_t)s_page[l] * 2 + sel) * a.page_size + m_slot[m]) * a.hkv + h) * D + u * E;
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

  collect(0);
  const bool single = tiles <= 1;
  if (single && members == 0) return;
  for (int m = tid; m < members; m += 256) atomicMin(&s_first[m_lead[m]], m_slot[m]);
  for (int b = 1; !single && b <= tiles; ++b) {
    collect(b);
    for (int m = tid; m < members; m += 256) atomicMin(&s_first[m_lead[m]], m_slot[m]);
  }
  const bool cached = single && 2 * members <= 32;     // at most two rows a 16-lane group, kept in registers

  for (int h = h0; h < h1; ++h) {
    const int buf = h & 1;
    float keep[2][2 * E];
    if (cached) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = grp + 16 * i;
        if (r < 2 * members) {
          row(m_tok[r >> 1], r & 1, h, keep[i]);
          take_max(r >> 1, r & 1, buf, keep[i]);
        }
      }
    } else {
      for (int b = 0; b <= (single ? 0 : tiles); ++b) {
        if (!single) collect(b);
        for (int r = grp; r < 2 * members; r += 16) {
          float x[2 * E];
          row(m_tok[r >> 1], r & 1, h, x);
          take_max(r >> 1, r & 1, buf, x);
        }
      }
    }
    if (tid == 0) s_grown = 0;
    __syncthreads();
    // ---- the blocks' new scales
    if (tid < 2 * kChunk) {
      const int l = tid >> 1, sel = tid & 1;
      s_amax[buf ^ 1][l][sel] = 0;
      if (s_lead[l] == l && s_first[l] >= 0 && s_first[l] < a.page_size) {
        uint8_t* sp = a.scale + ((int64_t)s_page[l] * 2 + sel) * a.hkv + h;
        int e = block_exp(s_amax[buf][l][sel]), old = e;
        if (s_first[l] > 0) {
          old = min((int)*sp - 127, 120);            // (120: the largest of a bf16 block)
          e = max(e, old);
          if (e > old) s_grown = 1;
        }
        s_exp[l][sel] = e;
        s_old[l][sel] = old;
        *sp = (uint8_t)(e + 127);
      } else {
        s_exp[l][sel] = s_old[l][sel] = 0;
      }
    }
    __syncthreads();
    // ---- the members' codes
    if (cached) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = grp + 16 * i;
        if (r < 2 * members) store(r >> 1, r & 1, h, keep[i]);
      }
    } else {
      for (int b = 0; b <= (single ? 0 : tiles); ++b) {
        if (!single) collect(b);
        for (int r = grp; r < 2 * members; r += 16) {
          float x[2 * E];
          row(m_tok[r >> 1], r & 1, h, x);
          store(r >> 1, r & 1, h, x);
        }
      }
    }
    // ---- tokens written before, where the scale grew
    if (s_grown) {
      for (int l = 0; l < cn; ++l)
        for (int sel = 0; sel < 2; ++sel) {
          const int by = s_old[l][sel] - s_exp[l][sel];
          if (by >= 0) continue;
          const float f = exp2i(max(by, -126));
          for (int t = grp; t < s_first[l]; t += 16) {
            uint8_t* d = a.kv + ((((int64_t)s_page[l] * 2 + sel) * a.page_size + t) * a.hkv + h) * D + u * (D / 16);
#pragma unroll
            for (int w = 0; w < D / 64; ++w) {
              typedef float f2 __attribute__((ext_vector_type(2)));
              const int c = *reinterpret_cast<const int*>(d + 4 * w);
              const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
              *reinterpret_cast<uint32_t*>(d + 4 * w) = codes4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
            }
          }
        }
    }
    __syncthreads();
  }
}

// grid.x = copy entry, grid.y = layer * 2 + K / V: the first len tokens' codes and,
// for any token at all, the page's scales of the source.
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
// the V planes only (from plane `first`).  HBM-bound: 1 byte read and 2 written a value.
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

// Entries of a workgroup and its share of the heads.  Few entries: four a workgroup
// and one KV head each, so that a decode step's rows spread over the CUs; many: 16 (a
// page's worth), and just enough shares to give every CU a few workgroups.
static int launch_append(AppendArgs& a, int dtype, int d, hipStream_t st) {
  a.chunk = a.n <= 1024 ? 4 : kChunk;
  const unsigned gx = (unsigned)((a.n + a.chunk - 1) / a.chunk);
  const unsigned gy = (unsigned)std::min<int64_t>(a.hkv, std::max<int64_t>(1, (2048 + gx - 1) / gx));
  const dim3 grid(gx, gy);
#define BE_APPEND(TY)                                                        \
  switch (d) {                                                               \
    case 64: append_kernel<TY, 64><<<grid, 256, 0, st>>>(a); break;          \
    case 128: append_kernel<TY, 128><<<grid, 256, 0, st>>>(a); break;        \
    default: append_kernel<TY, 256><<<grid, 256, 0, st>>>(a); break;         \
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
