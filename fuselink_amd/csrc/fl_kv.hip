// fl_kv.hip -- operators on KV pages held in 8 bits: storing keys and values into page records (flh_kv_store),
// attention over them (flh_kv_attend), the choice of pages by their key bounds (flh_kv_select) and the repacking of
// the tokens that attention has dwelt on (flh_kv_evict).  The records are bytes to the page movers of fl_copy.hip.
#include <hip/hip_runtime.h>

#include <cstring>
#include <type_traits>

#include "fl_device.h"
#include "fl_internal.h"
#include "fl_launch.h"
#include "fuselink_hip.h"

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

constexpr float kInf = __builtin_inff();
constexpr float kNan = __builtin_nanf("");
constexpr float kLeast = 0x1p-149f;      // stands for 0 as a factor of scores: what it multiplies is zero then, or -inf and stays so

// ------------------------------------------------------------------------------------------------
// records and sequences
// ------------------------------------------------------------------------------------------------
struct Cache {
  uint8_t* pages;
  uint64_t stride;
  uint32_t n_pages, T, H, D;
  uint64_t side, low, high, scales;   // byte offsets inside a record: V codes, bounds, scales
};

// Token counts come from device memory, so every use of them is clamped to what the host could check.
struct Seqs {
  const int32_t* starts;   // may be null: per tokens each
  const int32_t* lens;
  const int32_t* table;
  uint64_t table_stride;
  uint32_t width, n_seqs, n_tokens, per;
  int32_t* status;
};

// What no launch writes while it runs -- page tables, counts, scales of the records it reads -- at a uniform address:
// through the constant address space these are scalar loads, which do not queue behind the vector loads of the codes.
template <class T>
__device__ __forceinline__ T scalar_load(const T* p) {
  typedef const T __attribute__((address_space(4))) * P;
  return *(P)(uintptr_t)p;
}

__device__ __forceinline__ void report(int32_t* status) { *status = FLH_E_RANGE; }

__device__ __forceinline__ void seq_tokens(const Seqs& s, uint32_t b, uint32_t& first, uint32_t& n) {
  if (!s.starts) { first = b * s.per; n = s.per; return; }
  const int32_t lo = s.starts[b], hi = s.starts[b + 1];
  if (lo < 0 || hi < lo || (uint32_t)hi > s.n_tokens) { report(s.status); first = 0; n = 0; return; }
  first = (uint32_t)lo;
  n = (uint32_t)(hi - lo);
}

// the same for a sequence that the whole wavefront looks at
__device__ __forceinline__ void uniform_tokens(const Seqs& s, uint32_t b, uint32_t& first, uint32_t& n) {
  if (!s.starts) { first = b * s.per; n = s.per; return; }
  const int32_t lo = scalar_load(s.starts + b), hi = scalar_load(s.starts + b + 1);
  const bool ok = lo >= 0 && hi >= lo && (uint32_t)hi <= s.n_tokens;
  if (!ok) report(s.status);
  first = ok ? (uint32_t)lo : 0;
  n = ok ? (uint32_t)(hi - lo) : 0;
}
__device__ __forceinline__ uint32_t uniform_len(const Seqs& s, uint32_t T, uint32_t b) {
  const int32_t len = scalar_load(s.lens + b);
  const uint32_t most = s.width * T;   // (the host keeps it within 31 bits)
  if (len < 0 || (uint32_t)len > most) { report(s.status); return len < 0 ? 0u : most; }
  return (uint32_t)len;
}

// Item x of the sequences' items laid end to end: its sequence, which of that one's items it is, and the sequence's
// tokens.  A wavefront looks at 64 sequences at a time, all it needs to know of them loaded at once.  False if there
// are fewer items.  LONGEST: the sequences of 64 are laid out by length, the longest first, so that what is handed out
// last is short.  APPEND: tokens go behind the length, so a negative one (empty otherwise) leaves them no place.
struct Item { uint32_t b, local, first, n, len; };
template <bool LONGEST = false, bool APPEND = false, class Count>
__device__ __forceinline__ bool find_item(const Seqs& s, uint32_t T, uint32_t x, Count count, Item& it) {
  const int lane = threadIdx.x & 63;
  for (uint32_t base = 0; base < s.n_seqs; base += 64) {
    uint32_t first = 0, n = 0, len = 0, c = 0;
    if (base + lane < s.n_seqs) {
      const int32_t held = s.lens[base + lane];
      seq_tokens(s, base + lane, first, n);
      const uint32_t most = s.width * T;   // (the host keeps it within 31 bits)
      len = held < 0 ? 0u : (uint32_t)held > most ? most : (uint32_t)held;
      if ((uint32_t)held != len) report(s.status);
      if (APPEND && held < 0) n = 0;
      c = count(n, len);
    }
    uint32_t incl = wave_incl_sum_u32(c, lane);
    const uint32_t total = bcast_lane_u32(incl, 63);
    if (x < total) {
      if (LONGEST) {
        incl = c;
        const uint32_t cnt = s.n_seqs - base < 64 ? s.n_seqs - base : 64;
#pragma unroll 1
        for (uint32_t j = 0; j < cnt; ++j) {
          const uint32_t lj = bcast_lane_u32(len, (int)j), cj = bcast_lane_u32(c, (int)j);
          incl += lj > len || (lj == len && j < (uint32_t)lane) ? cj : 0;
        }
      }
      const int l = __builtin_ctzll(__ballot(incl > x && incl - c <= x));
      it.b = base + (uint32_t)l;
      it.local = x - (bcast_lane_u32(incl, l) - bcast_lane_u32(c, l));
      it.first = bcast_lane_u32(first, l);
      it.n = bcast_lane_u32(n, l);
      it.len = bcast_lane_u32(len, l);
      return true;
    }
    x -= total;
  }
  return false;
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// The larger of two as one instruction: the median with infinity.  (fmaxf also quiets each operand that may be a
// signalling NaN, which everything is that comes from a matrix instruction or another lane.)  A NaN gives way to a number.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, kInf); }

// the four lanes that share a column of a 16 x 16 result: l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float column_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// all lanes get the largest of the 64 (a row of 16 by DPP, the four rows as above)
__device__ __forceinline__ float wave_max_f32(float v) {
  v = fmaxf(v, __uint_as_float(dpp_u32<0xb1>(__float_as_uint(v))));    // quad_perm 1 0 3 2
  v = fmaxf(v, __uint_as_float(dpp_u32<0x4e>(__float_as_uint(v))));    // quad_perm 2 3 0 1
  v = fmaxf(v, __uint_as_float(dpp_u32<0x141>(__float_as_uint(v))));   // mirrored in 8
  v = fmaxf(v, __uint_as_float(dpp_u32<0x140>(__float_as_uint(v))));   // mirrored in 16
  return column_max(v);
}

// ------------------------------------------------------------------------------------------------
// e4m3 codes under a power-of-two scale
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// Smallest 2^e >= amax / 448 with e >= -126, 0 for amax = 0: 448 = 1.75 * 2^8, so the mantissa decides between two exponents.
__device__ __forceinline__ float block_scale(float amax) {
  if (!(amax > 0.f)) return 0.f;
  const uint32_t u = __float_as_uint(amax);
  const int x = (int)(u >> 23) - 127;
  int e = (u & 0x7fffffu) <= 0x600000u ? x - 8 : x - 7;
  if (e < -126 || u < 0x800000u) e = -126;
  return pow2f(e);
}
__device__ __forceinline__ float inverse(float s) {   // of a power of two, exact; 0 for 0
  return s > 0.f ? __uint_as_float((254u << 23) - __float_as_uint(s)) : 0.f;
}

// ------------------------------------------------------------------------------------------------
// blocks of tokens into records: new tokens behind those that a page holds (store), or chosen tokens of other
// records (evict)
// ------------------------------------------------------------------------------------------------
struct PackArgs {
  Cache c;
  Seqs s;
  // store
  const void* src[2];
  uint64_t token_stride[2], head_stride[2];   // in elements
  uint32_t vec;                               // 16-byte loads are aligned
  // evict
  Cache from;
  const int32_t* to_table;
  uint64_t to_stride;
  const int32_t* kept;
  uint64_t kept_stride;
  uint32_t per_seq, most;                     // most: tokens of a sequence that can be kept, by the budget and by the weights
};

// Eight neighbouring channels of a token as they lie in memory, and as numbers.
template <class E> struct Raw { uint32_t w[sizeof(E) * 2]; };
struct Code { uint32_t w[2]; float s; };

template <class E>
__device__ __forceinline__ void load_raw(Raw<E>& r, const E* p, bool vec) {
  constexpr int W = sizeof(E) * 2;
  if (vec) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint32_t*>(p) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[i + e] = x[e];
    }
  } else if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = reinterpret_cast<const uint16_t*>(p)[2 * i] | (uint32_t)reinterpret_cast<const uint16_t*>(p)[2 * i + 1] << 16;
  }
}
template <class E>
__device__ __forceinline__ float number(const Raw<E>& r, int i) {
  if constexpr (sizeof(E) == 4) return __uint_as_float(r.w[i]);
  else if constexpr (__is_same(E, __bf16)) return __uint_as_float(i & 1 ? r.w[i >> 1] & 0xffff0000u : r.w[i >> 1] << 16);
  else return (float)__builtin_bit_cast(h2, r.w[i >> 1])[i & 1];
}

// The largest magnitude as bits, which order as magnitudes do, two 16-bit ones to a word.  Infinities and NaN come
// above all that is finite: finite_amax() goes over the row again if there are any.
template <class E>
__device__ __forceinline__ void max_bits(uint32_t& m, const Raw<E>& r) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(E) * 2); ++i) {
    if constexpr (sizeof(E) == 4) { const uint32_t v = r.w[i] & 0x7fffffffu; m = v > m ? v : m; }
    else m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, m), __builtin_bit_cast(us2, r.w[i] & 0x7fff7fffu)));
  }
}
template <class E>
__device__ __forceinline__ float max_of_bits(uint32_t m) {
  if constexpr (sizeof(E) == 4) return __uint_as_float(m);
  const uint32_t v = (m & 0xffffu) > (m >> 16) ? m & 0xffffu : m >> 16;
  if constexpr (__is_same(E, __bf16)) return __uint_as_float(v << 16);
  else return (float)__builtin_bit_cast(h2, v)[0];
}
template <class E>
__device__ __forceinline__ float finite_amax(const Raw<E>& r) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) { const float v = fabsf(number(r, i)); m = v < kInf && v > m ? v : m; }
  return m;
}

// Eight channels as codes under a power-of-two scale.  The conversions divide by it and round to nearest even; what is
// not finite becomes NaN.
typedef short s2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float s) {
  s2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, s, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, s, true);
  return __builtin_bit_cast(uint32_t, r);
}
template <class E>
__device__ __forceinline__ u2 encode(const Raw<E>& x, float s) {
  u2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s2 r = {0, 0};
    if constexpr (__is_same(E, __bf16)) {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(b2, x.w[2 * i]), s, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(b2, x.w[2 * i + 1]), s, true);
      w[i] = __builtin_bit_cast(uint32_t, r);
    } else if constexpr (__is_same(E, _Float16)) {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(h2, x.w[2 * i]), s, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(h2, x.w[2 * i + 1]), s, true);
      w[i] = __builtin_bit_cast(uint32_t, r);
    } else {
      w[i] = encode4(__uint_as_float(x.w[4 * i]), __uint_as_float(x.w[4 * i + 1]), __uint_as_float(x.w[4 * i + 2]), __uint_as_float(x.w[4 * i + 3]), s);
    }
  }
  return w;
}
// codes under one scale as codes under another
__device__ __forceinline__ u2 recode(const uint32_t* w, float from, float to) {
  u2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i], from, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i], from, true);
    r[i] = encode4(a[0], a[1], b[0], b[1], to);
  }
  return r;
}
__device__ __forceinline__ u2 encode(const Code& x, float s) { return recode(x.w, x.s, s); }
__device__ __forceinline__ float amax_of(const Code& x) {   // (fmaxf passes over NaN)
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x.w[i], x.s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x.w[i], x.s, true);
    m = fmaxf(m, fmaxf(fmaxf(fabsf(a[0]), fabsf(a[1])), fmaxf(fabsf(b[0]), fabsf(b[1]))));
  }
  return m;
}
__device__ __forceinline__ h2 least(h2 a, h2 b) { return __builtin_elementwise_min(a, b); }
__device__ __forceinline__ h2 most(h2 a, h2 b) { return __builtin_elementwise_max(a, b); }
// over the four lanes l, l ^ 16, l ^ 32, l ^ 48
template <class F>
__device__ __forceinline__ h2 column_pair(h2 v, F f) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  u = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(h2, (uint32_t)r[0]), __builtin_bit_cast(h2, (uint32_t)r[1])));
  r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return f(__builtin_bit_cast(h2, (uint32_t)r[0]), __builtin_bit_cast(h2, (uint32_t)r[1]));
}

// W wavefronts pack K and V of one head of one page.  A lane holds 8 neighbouring channels of every RP-th token
// (RP = 64 / (D / 8) tokens at a time), so both the codes' rows and the channels' bounds come out of registers.  The
// largest magnitude of the new tokens fixes the scale, then the same rows become codes: every row is read once and stays
// in registers between the two, as it was loaded, ROWS of them a lane.  More than one wavefront exchange their largest
// magnitude and their bounds through shared memory.  In evict the rows are codes of other records under their own scales.
// Memory bounds it: 16 prompts of up to 4096 tokens, 8 heads of 128 channels in bf16, 267 MB in 62 us, 4.3 TB/s (a copy of 4 GiB: 4.5);
// 16 sequences cut back to 2048 tokens, 134 MB in 44 us, 3.0 TB/s, every row of 128 bytes from a place of its own, behind three
// loads that tell where.  (Here and at the kernels below inputs change from call to call and do not fit the caches together.)
template <class E, bool EVICT, int ROWS, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void fl_kv_pack(const PackArgs a) {
  warm_kernel_args(a);
  typedef typename std::conditional<EVICT, Code, Raw<E>>::type Row;
  constexpr bool kBoth = sizeof(Row) * ROWS * 2 <= (W == 16 ? 256 : 512);   // rows of K and of V fit the registers together
  __shared__ float part_max[2][W];
  __shared__ h2 part_low[W][32][4], part_high[W][32][4];
  const int lane = threadIdx.x & 63;
  const Cache& c = a.c;
  const uint32_t wave = uniform(threadIdx.x >> 6), part = W == 1 ? 0 : wave;
  const uint32_t h = W == 1 ? blockIdx.y * 4 + wave : blockIdx.y;
  if (h >= c.H) return;
  const uint32_t T = c.T, D = c.D;
  uint32_t b, j, first = 0, n, held;
  int32_t page;
  if constexpr (EVICT) {
    b = blockIdx.x / a.per_seq;
    j = blockIdx.x - b * a.per_seq;
    n = uniform_len(a.s, a.from.T, b);
    if (n > a.most) n = a.most;
    held = 0;
    if (j * T >= n) return;
    page = scalar_load(a.to_table + b * a.to_stride + j);
  } else {
    Item it;
    if (!find_item<false, true>(a.s, T, blockIdx.x, [&](uint32_t m, uint32_t l) { return m ? (l + m + T - 1) / T - l / T : 0; }, it)) return;
    b = it.b;
    first = it.first;
    n = it.n;
    held = it.len;
    j = it.local + held / T;
    if (j >= a.s.width) { if (lane == 0) report(a.s.status); return; }
    page = scalar_load(a.s.table + b * a.s.table_stride + j);
  }
  if (page < 0 || (uint32_t)page >= c.n_pages) { if (lane == 0) report(a.s.status); return; }
  const uint32_t at = j * T;                                   // position of the page's first slot
  const uint32_t old = held > at ? held - at : 0;              // slots that hold a token already
  const uint64_t end64 = (uint64_t)held + n - at;
  const uint32_t fill = end64 < T ? (uint32_t)end64 : T;       // slots that hold one afterwards
  uint8_t* rec = c.pages + (uint64_t)page * c.stride;

  const uint32_t CG = D >> 3, RP = 64 / CG, grp = (uint32_t)lane / CG, cg = (uint32_t)lane - grp * CG;
  const bool on = grp < RP;

  // Rows (i * W + part) * RP + grp: new tokens (evict: all of them), 0 elsewhere.  sides: 1 K, 2 V, 3 both
  Row x[2][ROWS];
  const auto load = [&](const int sides) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const uint32_t r = (i * W + part) * RP + grp;
#pragma unroll
      for (int side = 0; side < 2; ++side)
        if (sides >> side & 1) x[side][i] = Row{};
      if (!on || r >= fill || r < old) continue;
      if constexpr (EVICT) {
        const int32_t pos = a.kept[(b * (uint64_t)c.H + h) * a.kept_stride + at + r];
        const uint32_t slot = (uint32_t)pos / a.from.T;
        const int32_t pg = pos >= 0 && slot < a.s.width ? a.s.table[b * a.s.table_stride + slot] : -1;
        if (pg < 0 || (uint32_t)pg >= a.from.n_pages) { report(a.s.status); continue; }
        const uint8_t* f = a.from.pages + (uint64_t)pg * a.from.stride;
        const uint64_t off = ((uint64_t)h * a.from.T + ((uint32_t)pos - slot * a.from.T)) * D + cg * 8;
        const u2 s = *reinterpret_cast<const u2*>(f + a.from.scales + 8 * h);
#pragma unroll
        for (int side = 0; side < 2; ++side)
          if (sides >> side & 1) {
            const u2 w = *reinterpret_cast<const u2*>(f + side * a.from.side + off);
            x[side][i] = Code{{w[0], w[1]}, __uint_as_float(s[side])};
          }
      } else {
#pragma unroll
        for (int side = 0; side < 2; ++side)
          if (sides >> side & 1)
            load_raw<E>(x[side][i], reinterpret_cast<const E*>(a.src[side]) + (uint64_t)(first + at + r - held) * a.token_stride[side] + h * a.head_stride[side] + cg * 8, a.vec);
      }
    }
  };
  const auto pack = [&](const int side) {
    float* scale_at = reinterpret_cast<float*>(rec + c.scales) + 2 * h + side;
    const float s_old = !EVICT && old ? *scale_at : 0.f;
    float amax = 0.f;
    if (!kBoth) load(1 << side);
    if constexpr (EVICT) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) amax = fmaxf(amax, amax_of(x[side][i]));
    } else {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) max_bits<E>(bits, x[side][i]);
      amax = max_of_bits<E>(bits);
      if (__ballot(!(amax < kInf))) {
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) amax = fmaxf(amax, finite_amax<E>(x[side][i]));
      }
    }
    amax = wave_max_f32(amax);
    if constexpr (W > 1) {
      if (lane == 0) part_max[side][part] = amax;
      __syncthreads();
      amax = wave_max_f32(part_max[side][lane & (W - 1)]);
    }
    const float s = fmaxf(s_old, block_scale(amax));
    const bool grown = old && s != s_old;
    h2 lo[4], hi[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { lo[e] = h2{(_Float16)kInf, (_Float16)kInf}; hi[e] = -lo[e]; }
    uint8_t* codes = rec + side * c.side + (uint64_t)h * T * D;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const uint32_t r = (i * W + part) * RP + grp;
      if (!on || r >= T) continue;
      u2* row = reinterpret_cast<u2*>(codes + r * D + cg * 8);
      u2 w;
      if (r < old) {
        if (side == 1 && !grown) continue;
        w = *row;
        if (grown) { const uint32_t t[2] = {w[0], w[1]}; w = recode(t, s_old, s); }
      } else {
        w = encode(x[side][i], s);
      }
      if (r < old ? grown : (r < fill || !old)) *row = w;   // slots behind the tokens of a page that this call opens are zero
      if (side == 0 && r < fill) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const h2 v = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e >> 1], 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e >> 1], 1.f, false);
          lo[e] = least(lo[e], v);
          hi[e] = most(hi[e], v);
        }
      }
    }
    if (lane == 0 && part == 0) *scale_at = s;
    if (side == 1) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (CG == 16) {
        lo[e] = column_pair(lo[e], least);
        hi[e] = column_pair(hi[e], most);
      } else {
        const uint32_t l0 = __builtin_bit_cast(uint32_t, lo[e]), u0 = __builtin_bit_cast(uint32_t, hi[e]);
        for (uint32_t k = 1; k < RP; ++k) {
          lo[e] = least(lo[e], __builtin_bit_cast(h2, __shfl((int)l0, (int)(cg + k * CG))));
          hi[e] = most(hi[e], __builtin_bit_cast(h2, __shfl((int)u0, (int)(cg + k * CG))));
        }
      }
    }
    if constexpr (W > 1) {
      if (lane < (int)CG)
#pragma unroll
        for (int e = 0; e < 4; ++e) { part_low[part][lane][e] = lo[e]; part_high[part][lane][e] = hi[e]; }
      __syncthreads();
      if (part == 0 && lane < (int)CG)
#pragma unroll 3
        for (int k = 1; k < W; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) { lo[e] = least(lo[e], part_low[k][lane][e]); hi[e] = most(hi[e], part_high[k][lane][e]); }
    }
    if (part == 0 && lane < (int)CG) {
      u2 wl = {0, 0}, wh = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float l = (float)lo[e >> 1][e & 1], u = (float)hi[e >> 1][e & 1];
        const int li = l <= u ? (int)floorf(l * 0.25f) : 0, ui = l <= u ? (int)ceilf(u * 0.25f) : 0;   // (not so: no finite one)
        wl[e >> 2] |= (uint32_t)(li & 0xff) << (8 * (e & 3));
        wh[e >> 2] |= (uint32_t)(ui & 0xff) << (8 * (e & 3));
      }
      *reinterpret_cast<u2*>(rec + c.low + (uint64_t)h * D + cg * 8) = wl;
      *reinterpret_cast<u2*>(rec + c.high + (uint64_t)h * D + cg * 8) = wh;
    }
  };

  if (kBoth) load(3);
  pack(0);
  pack(1);
}

// ------------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------------
struct AttendArgs {
  Cache c;
  Seqs s;
  const void* q;
  void* out;
  float* lse;                 // natural logarithm, for the caller (may be null)
  float* lse2;                // [n_tokens][H G] base 2, for the weights (may be null)
  uint64_t q_token, q_head, o_token, o_head;
  uint32_t G, tiles_x, splits;
  uint32_t per_page, per_page_inv;   // tiles of 16 tokens to a page; 2^32 over it, rounded up: exact for the 2^27 tiles there can be
  float scale2;               // |scale| * log2(e); the queries carry the sign
  uint32_t flip;              // sign bits of two 16-bit numbers, or 0
  uint32_t causal, q_vec, o_vec;
  const int32_t* sel;         // [n_tokens][H][count] pages of every query token, or null
  uint32_t count;
  float* part_o;              // [splits][n_tokens * H * G][D]
  float* part_l;              // [splits][n_tokens * H * G]
  const float* w_in;          // [n_seqs][H][w_stride]
  float* w_out;
  uint64_t wi_seq, wi_head, wo_seq, wo_head;
  uint32_t w_width;
};

template <class E> struct Frag;
template <> struct Frag<_Float16> {
  typedef h8 v8;
  template <bool HI> static __device__ __forceinline__ h2 pk(uint32_t w) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI); }
  static __device__ __forceinline__ f4 mfma(v8 a, v8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<__bf16> {
  typedef b8 v8;
  template <bool HI> static __device__ __forceinline__ b2 pk(uint32_t w) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI); }
  static __device__ __forceinline__ f4 mfma(v8 a, v8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
// 8 codes as 8 numbers of the query's type: e4m3 fits both exactly
template <class E>
__device__ __forceinline__ typename Frag<E>::v8 codes8(uint32_t w0, uint32_t w1) {
  typename Frag<E>::v8 r;
  const auto a = Frag<E>::template pk<false>(w0), b = Frag<E>::template pk<true>(w0), c = Frag<E>::template pk<false>(w1), d = Frag<E>::template pk<true>(w1);
  r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1]; r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <class E>
__device__ __forceinline__ typename Frag<E>::v8 load_q8(const E* p, bool ok, bool vec) {
  typename Frag<E>::v8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (E)0.f;
  if (ok) {
    if (vec) {
      r = *reinterpret_cast<const typename Frag<E>::v8*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = p[i];
    }
  }
  return r;
}

template <class E>
__device__ __forceinline__ typename Frag<E>::v8 flipped(typename Frag<E>::v8 x, uint32_t flip) {
  u32x4 w = __builtin_bit_cast(u32x4, x);
  w ^= flip;
  return __builtin_bit_cast(typename Frag<E>::v8, w);
}

// What a wavefront carries for its NQ x 16 rows: O^T in units of 2^(ev - 127), each lane's part of the rows' sums of
// exp2(x - ref), the maximum that ref = top - 8 comes from.  fresh: a row that may see keys has not seen
// one.  elow: ev does not fall below it.
template <int NQ, int VJ>
struct Rows {
  f4 o[NQ][VJ];
  float top[NQ], ref[NQ], l[NQ];
  int ev, elow;
  bool fresh;
};
template <int NQ, int VJ>
__device__ __forceinline__ void clear(Rows<NQ, VJ>& r, const uint32_t (&lim)[NQ], uint32_t k0) {
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    r.top[q] = lim[q] > k0 ? -kInf : 0.f;
    r.ref[q] = r.l[q] = 0.f;
#pragma unroll
    for (int j = 0; j < VJ; ++j) r.o[q][j] = f4{0.f, 0.f, 0.f, 0.f};
  }
  r.ev = r.elow = 0;
  r.fresh = true;
}

// the exponent field of a value scale, 0 for none
__device__ __forceinline__ int scale_bits(float v) { return (int)(uniform(__float_as_uint(v)) >> 23); }
// Value scales of a step's two tiles more than 2^6 apart: the smaller one's probabilities would lose their bits to the larger
// one's unit, for rows, too, that do not see the larger.  The smaller tile is then left out, and taken alone behind all others.
__device__ __forceinline__ bool apart(int x0, int x1) { return x0 && x1 && (uint32_t)(x0 - x1 + 6) > 12; }

// One step of the softmax: scores of 32 keys (two tiles under K scales kc0 and kc1, base 2, and value scales v0 and v1) to
// probabilities and their sums.
//
// A row's probabilities are exp2(x - ref) with a reference that follows its maximum only when one of them would pass 2^15,
// which is seen from the rounded ones themselves, two to a word; the maximum proper is taken in that case only.  The
// tiles' value scales go into the probabilities as powers of two of the scale that O counts in (exact, and free in the
// exponent), so that V's codes meet them as they are.  That scale is the larger of the two blocks', kept while it stays
// within 2^6 below; it never falls more than 2^60 below the largest so far, or what O holds would overflow (the other tile of
// a step is at most 2^6 smaller, see apart()).  The sums
// take the probabilities before they are rounded: logarithms and weights are 32 bits wide and come from them.
template <int NQ, int VJ>
__device__ __forceinline__ void soften(Rows<NQ, VJ>& r, const f4 (&s)[NQ][2], float kc0, float kc1, float v0, float v1, h8 (&pf)[NQ]) {
  const int x0 = scale_bits(v0), x1 = scale_bits(v1), xm = x0 > x1 ? x0 : x1, xt = xm > r.elow ? xm : r.elow;
  const int enew = xm > 0 && !(xt <= r.ev && xt + 6 >= r.ev) ? xt : r.ev;
  const int d0 = x0 - enew < -64 ? -64 : x0 - enew, d1 = x1 - enew < -64 ? -64 : x1 - enew;   // (a block of zeros: the least)
  const float e0 = (float)d0, e1 = (float)d1;
  if (enew != r.ev) {
    asm volatile("");
    const int dv = r.ev - enew;
    const float fv = r.ev == 0 ? 1.f : dv < -126 ? 0.f : pow2f(dv);
    r.ev = enew;
    if (enew - 60 > r.elow) r.elow = enew - 60;
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int j = 0; j < VJ; ++j) r.o[q][j] *= fv;
  }
  const float u0 = pow2f(-d0), u1 = pow2f(-d1);
  bool none = false;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    float sum;
    uint32_t high;
    const auto exponentials = [&]() {
      const float r0 = e0 - r.ref[q], r1 = e1 - r.ref[q];
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = exp2_fast(__builtin_fmaf(s[q][i >> 2][i & 3], i < 4 ? kc0 : kc1, i < 4 ? r0 : r1));
        pf[q][i] = (_Float16)p[i];
      }
      sum = ((p[0] + p[1]) + (p[2] + p[3])) * u0 + ((p[4] + p[5]) + (p[6] + p[7])) * u1;
      const u32x4 w = __builtin_bit_cast(u32x4, pf[q]);
      const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];   // (a bit cast of a vector's element takes the first one's bits)
      const us2 m = __builtin_elementwise_max(__builtin_elementwise_max(__builtin_bit_cast(us2, w0), __builtin_bit_cast(us2, w1)),
                                              __builtin_elementwise_max(__builtin_bit_cast(us2, w2), __builtin_bit_cast(us2, w3)));
      high = __builtin_bit_cast(uint32_t, m) + 0x08000800u;   // bit 15 of a half: 2^15 or more, or no number
    };
    exponentials();
    if (r.fresh || __ballot((high & 0x80008000u) != 0)) {
      asm volatile("");
      // (where all are NaN this is infinity, and the row's sum NaN one way or the other)
      const float m0 = larger(larger(s[q][0][0], s[q][0][1]), larger(s[q][0][2], s[q][0][3]));
      const float m1 = larger(larger(s[q][1][0], s[q][1][1]), larger(s[q][1][2], s[q][1][3]));
      const float t = larger(r.top[q], column_max(larger(m0 * kc0, m1 * kc1))), f = r.top[q] == -kInf ? 0.f : exp2_fast(r.top[q] - t);
      r.top[q] = t;
      r.ref[q] = t == -kInf ? 0.f : t - 8.f;
      none |= t == -kInf;
      r.l[q] *= f;
#pragma unroll
      for (int j = 0; j < VJ; ++j) r.o[q][j] *= f;
      exponentials();
    }
    r.l[q] += sum;
  }
  if (r.fresh) r.fresh = __ballot(none) != 0;
}

// four codes of each of two tokens as pairs: v[j] gets (first token's, second's) of code j
__device__ __forceinline__ void interleave(uint32_t w0, uint32_t w1, h2 (&v)[4]) {
  const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400u), hi = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
  v[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  v[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  v[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  v[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
}
// codes of NaN become zero; what was found is or-ed into `seen`
__device__ __forceinline__ uint32_t without_nan(uint32_t w, uint32_t& seen) {
  const uint32_t nan = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;   // bytes whose magnitude is 0x7f
  seen |= nan;
  return w & ~((nan >> 7) * 0xffu);
}

// eight dims of row r's result, to the output or, if there are splits, to this split's part of the workspace
template <class E>
__device__ __forceinline__ void emit8(const AttendArgs& a, uint32_t split, uint32_t first, uint32_t h, uint32_t r, float mm, float ll, const float* v, uint32_t d, bool head) {
  const uint32_t H = a.c.H, G = a.G, D = a.c.D, i = r / G;
  const uint64_t tok = first + i, hq = h * G + (r - i * G);
  const float lg = ll > 0.f ? mm + __builtin_amdgcn_logf(ll) : (ll == 0.f ? -kInf : kNan);
  if (a.splits > 1) {
    const uint64_t at = (uint64_t)split * a.s.n_tokens * H * G + tok * H * G + hq;
    if (head) a.part_l[at] = lg;
    if (d < D) {
#pragma unroll
      for (int e = 0; e < 8; e += 4) *reinterpret_cast<f4*>(a.part_o + at * D + d + e) = f4{v[e], v[e + 1], v[e + 2], v[e + 3]};
    }
  } else {
    if (head) {
      if (a.lse) a.lse[tok * H * G + hq] = lg * 0.6931471805599453f;
      if (a.lse2) a.lse2[tok * H * G + hq] = lg;
    }
    E* p = reinterpret_cast<E*>(a.out) + tok * a.o_token + hq * a.o_head + d;
    if (d < D) {
      typename Frag<E>::v8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (E)v[e];
      if (a.o_vec) {
        *reinterpret_cast<typename Frag<E>::v8*>(p) = y;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = y[e];
      }
    }
  }
}

// Softmax and both products in one pass over the keys.  S^T = K Q^T and O^T = V^T P^T on 16 x 16 x 32 matrix
// instructions: a lane's column is one query row in both, so the row's maximum, sum and rescaling need no data from
// other rows, and S^T leaves the first product in the very lanes and order in which the second one wants P^T if the
// 32 keys of a step are numbered (two tiles of 16) x (four lane groups) x 4 -- an order that sums do not see.  K and V
// come as rows of codes straight into registers; V's bytes are interleaved token against token on the way to pairs.
// P is rounded to 16-bit floats (11 bits of mantissa) at 2^8 to 2^15 times its value relative to the row's largest and, for
// value scales below the one O counts in, at up to 2^-12 of that: normal down to 2^-22 of the largest, and to 2^-10 at worst.  Sums, references and accumulators
// are 32 bits wide and rarely rescaled.  Memory bounds it for up to 16 rows: 16 sequences of 131072 tokens, 8 heads of 128 channels,
// 4.3 GB in 720 us, 6.0 TB/s (a sum over 4 GiB: 6.1); 32 of up to 4096, 172 MB in 47 us, 3.7 TB/s, where the launch's
// start and the longest sequence show; 201 tokens 9 us, 4 of them the launch's.
template <class E, int DP, int NQ, bool SEL>
__global__ __launch_bounds__(256, DP == 256 ? 1 : NQ == 1 && DP == 128 ? 3 : 2) void fl_kv_attend(const AttendArgs a) {
  warm_kernel_args(a);
  constexpr int KK = DP / 32, KW = DP / 16, VJ = DP / 16, VW = DP / 64;
  constexpr uint32_t KVW = 4, TR = 16 * NQ;
  typedef typename Frag<E>::v8 v8;
  __shared__ float sm_o[KVW * 16 * NQ * (DP + 4)];
  __shared__ float sm_m[KVW * 16 * NQ], sm_l[KVW * 16 * NQ];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const uint32_t wave = uniform(threadIdx.x >> 6), H = a.c.H, G = a.G, T = a.c.T, D = a.c.D;
  const uint32_t h = blockIdx.x % H, rest = blockIdx.x / H, split = rest / a.tiles_x, x = rest - split * a.tiles_x;

  uint32_t tile, r0, rows, tok0 = 0;
  Item it;
  if constexpr (SEL) {
    const uint32_t per = (G + TR - 1) / TR, t = x / per;
    if (!find_item(a.s, T, t, [](uint32_t m, uint32_t) { return m; }, it)) return;
    tok0 = it.local;
    tile = x - t * per;
  } else {
    if (!find_item(a.s, T, x, [&](uint32_t m, uint32_t) { return (m * G + TR - 1) / TR; }, it)) return;
    tile = it.local;
  }
  const uint32_t b = it.b, first = it.first, n = it.n, len = it.len;
  // rows of this workgroup: (query token, head of the group), tokens first
  if constexpr (SEL) { r0 = tok0 * G + tile * TR; rows = (tok0 + 1) * G; } else { r0 = tile * TR; rows = n * G; }
  const auto limit = [&](uint32_t r) -> uint32_t {   // keys that row r sees
    if (r >= rows) return 0;
    if (!a.causal) return len;
    const int64_t l = (int64_t)len - n + r / G + 1;
    return l > 0 ? (uint32_t)l : 0;
  };
  const uint32_t last_row = r0 + 16 * NQ - 1 < rows ? r0 + 16 * NQ - 1 : rows - 1;
  const uint32_t l_min = uniform(r0 < rows ? limit(r0) : 0), l_max = uniform(r0 < rows ? limit(last_row) : 0);

  v8 qf[NQ][KK];
  uint32_t lim[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const uint32_t r = r0 + q * 16 + c;
    lim[q] = limit(r);
    const uint32_t i = r / G;
    const E* p = reinterpret_cast<const E*>(a.q) + (uint64_t)(first + i) * a.q_token + (uint64_t)(h * G + (r - i * G)) * a.q_head;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      const uint32_t d = g * (DP / 4) + k * 8;
      qf[q][k] = flipped<E>(load_q8<E>(p + d, r < rows && d < D, a.q_vec), a.flip);
    }
  }

  // The keys of this split, in steps of 32.  The host knows how many splits there are, the device how long the sequence
  // is: every split takes an equal share of it in whole rounds of the workgroup's wavefronts.  Of a list of pages no more
  // entries than the sequence has pages (23 sequences of 3 tokens with lists of 196: 68 us without this).
  const uint32_t pages = (l_max + T - 1) / T, space = SEL ? (a.count < pages ? a.count : pages) * T : l_max, share = KVW * 32 * ((space + a.splits * KVW * 32 - 1) / (a.splits * KVW * 32));
  const uint64_t k0_64 = (uint64_t)split * share;
  const uint32_t k0 = k0_64 < space ? (uint32_t)k0_64 : space, k1 = share < space - k0 ? k0 + share : space;
  Rows<NQ, VJ> st;
  clear(st, lim, SEL ? 0 : k0);
  const int32_t* table = a.s.table + b * a.s.table_stride;
  const int32_t* sel = SEL ? a.sel + ((uint64_t)(first + tok0) * H + h) * a.count : nullptr;
  const uint32_t head_off = h * T * D;
  uint32_t k_lane[KW / 4], v_lane[4];   // this lane's bytes of a tile; lanes beyond D read what no one multiplies or writes
#pragma unroll
  for (int i = 0; i < KW / 4; ++i) k_lane[i] = c * D + (g * (DP / 4) + 16 * i < D ? g * (DP / 4) + 16 * i : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) v_lane[i] = (4 * g + i) * D + ((uint32_t)(c * VJ) < D ? c * VJ : 0);
  uint32_t bad = 0, nan_steps = 0, left_out = 0;

  // Four steps are under way at a time: the choice of a page (a load if pages were selected), its number, the codes and
  // scales, the sums.  Nothing in the first three branches: past the end they look at the last tile again.
  struct Choice { uint32_t at[2], slot[2]; bool ok[2]; };
  struct Where { uint32_t pos[2], page[2], off[2]; bool ok[2]; };
  const uint32_t last_tile = (k1 - 1) >> 4;   // (used when there are keys)
  const auto choose = [&](uint32_t k) {
    Choice r;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t tv = (k >> 4) + t, tl = tv < last_tile ? tv : last_tile, j = a.per_page == 1 ? tl : __umulhi(tl, a.per_page_inv);
      r.slot[t] = (tl - j * a.per_page) << 4;
      r.at[t] = SEL ? (uint32_t)scalar_load(sel + j) : j;
      r.ok[t] = tv <= last_tile;
    }
    return r;
  };
  const auto look_up = [&](const Choice& r) {
    Where w;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t at = r.at[t];
      w.ok[t] = r.ok[t];
      if (SEL) {
        w.ok[t] = w.ok[t] && at < a.s.width;
        at = at < a.s.width ? at : 0;
      }
      w.pos[t] = at * T + r.slot[t];
      w.ok[t] = w.ok[t] && w.pos[t] < l_max;
      w.off[t] = head_off + r.slot[t] * D;
      w.page[t] = (uint32_t)scalar_load(table + at);
    }
    return w;
  };
  struct Stage { uint32_t kw[2][KW], vw[8][VW], pos[2]; float ks[2], vs[2]; bool ok[2]; };
  const auto fetch = [&](Stage& s, const Where& w) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool there = w.page[t] < a.c.n_pages;
      bad |= w.ok[t] && !there ? 1 : 0;
      s.pos[t] = w.pos[t];
      s.ok[t] = w.ok[t] && there;
      const uint8_t* rec = a.c.pages + (uint64_t)(there ? w.page[t] : 0) * a.c.stride;
      const float* sc = reinterpret_cast<const float*>(rec + a.c.scales) + 2 * h;
      s.ks[t] = scalar_load(sc);
      s.vs[t] = scalar_load(sc + 1);
      const uint8_t *base = rec + w.off[t], *vb = base + a.c.side;
      asm("" : "+s"(base), "+s"(vb));   // scalar bases, so that a load's address is one register of this lane
#pragma unroll
      for (int i = 0; i < KW / 4; ++i) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(base + k_lane[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s.kw[t][4 * i + e] = x[e];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(vb + v_lane[i]);
        if constexpr (VW == 1) s.vw[4 * t + i][0] = p[0];
        else if constexpr (VW == 2) { const u2 x = *reinterpret_cast<const u2*>(p); s.vw[4 * t + i][0] = x[0]; s.vw[4 * t + i][1] = x[1]; }
        else {
          const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) s.vw[4 * t + i][e] = x[e];
        }
      }
    }
  };
  const auto work = [&](Stage& x) {
    if (!x.ok[0] && !x.ok[1]) return;
    if (const int x0 = scale_bits(x.vs[0]), x1 = scale_bits(x.vs[1]); x.ok[0] && x.ok[1] && apart(x0, x1)) {
      asm volatile("");
      x.ok[x0 < x1 ? 0 : 1] = false;
      left_out = 1;
    }
    const bool masked = !x.ok[0] || !x.ok[1] || x.pos[0] + 16 > l_min || x.pos[1] + 16 > l_min;

    f4 s[NQ][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[q][t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const v8 kf = codes8<E>(x.kw[t][2 * kk], x.kw[t][2 * kk + 1]);
#pragma unroll
        for (int q = 0; q < NQ; ++q) s[q][t] = Frag<E>::mfma(kf, qf[q][kk], s[q][t]);
      }
    }

    if (masked) {
      asm volatile("");   // a branch, not selects on every step's way
      // A row that does not see a key must not see its value either, and 0 * NaN is NaN: values nobody sees become
      // zero, and a NaN that some rows see goes into their sums by hand.
      uint32_t seen_nan = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t p = x.pos[t] + 4 * g + i;
          const bool keep = x.ok[t] && p < l_max;
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            if (!(x.ok[t] && p < lim[q])) s[q][t][i] = -kInf;
#pragma unroll
          for (int e = 0; e < VW; ++e) x.vw[4 * t + i][e] = without_nan(keep ? x.vw[4 * t + i][e] : 0, seen_nan);
        }
      if (__ballot(seen_nan != 0)) nan_steps = 1;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (!x.ok[t]) x.ks[t] = x.vs[t] = 0.f;   // anyone's: O's scale must not follow them
    }

    const float kc0 = fmaxf(x.ks[0] * a.scale2, kLeast), kc1 = fmaxf(x.ks[1] * a.scale2, kLeast);
    h8 pf[NQ];
    soften(st, s, kc0, kc1, x.vs[0], x.vs[1], pf);

#pragma unroll
    for (int e = 0; e < VW; ++e) {
      h8 vf[4];
#pragma unroll
      for (int pr = 0; pr < 4; ++pr) {
        h2 v[4];
        interleave(x.vw[2 * pr][e], x.vw[2 * pr + 1][e], v);
#pragma unroll
        for (int j = 0; j < 4; ++j) { vf[j][2 * pr] = v[j][0]; vf[j][2 * pr + 1] = v[j][1]; }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < NQ; ++q) st.o[q][4 * e + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[j], pf[q], st.o[q][4 * e + j], 0, 0, 0);
    }
  };

  {
    constexpr uint32_t kStep = 32 * KVW;
    uint32_t k = k0 + (wave * 32);
    if (k < k1) {
      // The fetch is unconditional: behind a branch, the wait for this step's codes would have to cover the next ones'
      // as well.
      Stage s0, s1;
      Where w = look_up(choose(k));
      Choice r = choose(k + kStep);
      fetch(s0, w);
      w = look_up(r);
      r = choose(k + 2 * kStep);
      for (;;) {
        fetch(s1, w);
        w = look_up(r);
        r = choose(k + 3 * kStep);
        work(s0);
        k += kStep;
        if (k >= k1) break;
        fetch(s0, w);
        w = look_up(r);
        r = choose(k + 3 * kStep);
        work(s1);
        k += kStep;
        if (k >= k1) break;
      }
    }
    if (left_out) {   // the smaller tiles of steps whose value scales lie apart
      for (k = k0 + (wave * 32); k < k1; k += kStep) {
        Stage s;
        fetch(s, look_up(choose(k)));
        const int x0 = scale_bits(s.vs[0]), x1 = scale_bits(s.vs[1]);
        if (!s.ok[0] || !s.ok[1] || !apart(x0, x1)) continue;
        s.ok[x0 < x1 ? 1 : 0] = false;
        work(s);
      }
    }
    if (nan_steps) {   // a NaN value that not every row of the tile sees: into the sums of those that do
      for (k = k0 + (wave * 32); k < k1; k += kStep) {
        Where w = look_up(choose(k));
#pragma unroll
        for (int t = 0; t < 2; ++t) w.ok[t] = w.ok[t] && w.page[t] < a.c.n_pages;
        if (!left_out && w.ok[0] && w.ok[1] && w.pos[0] + 16 <= l_min && w.pos[1] + 16 <= l_min) continue;
        for (int t = 0; t < 2; ++t) {
          if (!w.ok[t]) continue;
          const uint8_t* base = a.c.pages + (uint64_t)w.page[t] * a.c.stride + a.c.side + w.off[t];
          for (uint32_t kx = 0; kx < 16 && w.pos[t] + kx < l_max; ++kx)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < VJ; ++j) {
                const uint32_t d = (4 * g + i) * VJ + j;
                const bool nan = d < D && (base[kx * D + d] & 0x7f) == 0x7f;
#pragma unroll
                for (int q = 0; q < NQ; ++q) st.o[q][j][i] += nan && w.pos[t] + kx < lim[q] ? kNan : 0.f;
              }
        }
      }
    }
  }
  if (bad && lane == 0) report(a.s.status);
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    // O is the sum l times an average of values, in units of their scale, and may pass an end of the range that the average
    // keeps within: the unit follows behind the power of two of l, which the factors below give back.  (One change of the
    // exponent in place of two products: the selected form spills 50 scalars more into its loop, 64 pages 15.0 -> 16.9 us.)
    const float l = column_sum(st.l[q]), unit = st.ev > 0 ? pow2f(st.ev - 127) : 0.f, down = pow2f(-__builtin_amdgcn_frexp_expf(l));
    const int w = (int)wave * 16 * NQ + q * 16 + c;
    if (g == 0) { sm_m[w] = l == 0.f ? -kInf : st.ref[q]; sm_l[w] = l; }
    float* p = sm_o + w * (DP + 4) + g * 4 * VJ;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VJ; ++j) p[i * VJ + j] = st.o[q][j][i] * down * unit;
  }
  __syncthreads();
  for (uint32_t u = threadIdx.x; u < 16 * NQ * (DP / 8); u += 256) {
    const uint32_t rr = u / (DP / 8), d = (u - rr * (DP / 8)) * 8, r = r0 + rr;
    if (r >= rows || d >= D) continue;
    float mm = -kInf, ll = 0.f, v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (uint32_t w = 0; w < KVW; ++w) mm = fmaxf(mm, sm_m[w * 16 * NQ + rr]);
    float share[KVW];
#pragma unroll
    for (uint32_t w = 0; w < KVW; ++w) {
      const float l = sm_l[w * 16 * NQ + rr], f = mm == -kInf ? 1.f : exp2_fast(sm_m[w * 16 * NQ + rr] - mm);
      ll += l * f;
      share[w] = __builtin_amdgcn_ldexpf(f, __builtin_amdgcn_frexp_expf(l));
    }
    const float f = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
    for (uint32_t w = 0; w < KVW; ++w) {
      const float* p = sm_o + (w * 16 * NQ + rr) * (DP + 4) + d;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += p[e] * (share[w] * f);
    }
    emit8<E>(a, split, first, h, r, mm, ll, v, d, d == 0);
  }
}

// The same for many rows to a key-value head, where the matrix instructions and the exponentials bound it: each of the
// four wavefronts owns 32 rows and all walk over the keys together, 64 at a time.  Every wavefront looks up, fetches and
// converts one tile of 16 and leaves it in shared memory as the operands of the matrix instructions, with its scales, so
// that a code is converted once for 128 rows instead of once for 32 and the registers hold a quarter of the codes on
// their way.  Two barriers to 64 keys; the three workgroups of a compute unit fill each other's waits.  4 sequences of up
// to 16384 tokens, 1024 of them new, 32 query heads of 128: 632 GFLOP in 812 us, 780 TFLOP/s (a library product of 8192^3
// in bf16: 1271).  Neither kind of instruction bounds it: matrix instructions keep their pipes busy for 36 % of a SIMD's cycles,
// vector instructions (exponentials, conversions, packing) theirs for 53 %, and they take turns more than they overlap -- in
// a wavefront the softmax stands between the two products, and the barriers keep the four in step.
template <class E, int DP>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 3) void fl_kv_attend_rows(const AttendArgs a) {
  warm_kernel_args(a);
  constexpr int NQ = 2, KK = DP / 32, KW = DP / 16, VJ = DP / 16, VW = DP / 64;
  constexpr uint32_t TR = 64 * NQ;
  typedef typename Frag<E>::v8 v8;
  __shared__ v8 sm_k[4 * KK * 64];                     // [tile][kk][lane]
  __shared__ h8 sm_v[2 * VJ * 64];                     // [pair of tiles][j][lane]
  __shared__ f4 sm_tile[4];                            // K scale * scale2, V scale, there is such a tile
  __shared__ float sm_scale[4];                        // V scales of the next 64 keys' tiles, 0 for none
  __shared__ uint32_t sm_nan, sm_left_out;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const uint32_t wave = uniform(threadIdx.x >> 6), H = a.c.H, G = a.G, T = a.c.T, D = a.c.D;
  const uint32_t h = blockIdx.x % H, rest = blockIdx.x / H, split = rest / a.tiles_x, x = rest - split * a.tiles_x;
  Item it;
  if (!find_item<true>(a.s, T, x, [&](uint32_t m, uint32_t) { return (m * G + TR - 1) / TR; }, it)) return;
  const uint32_t b = it.b, first = it.first, n = it.n, len = it.len, r0 = it.local * TR, rows = n * G, wr0 = r0 + wave * 16 * NQ;
  const auto limit = [&](uint32_t r) -> uint32_t {   // keys that row r sees
    if (r >= rows) return 0;
    if (!a.causal) return len;
    const int64_t l = (int64_t)len - n + r / G + 1;
    return l > 0 ? (uint32_t)l : 0;
  };
  const auto last_of = [&](uint32_t from, uint32_t cnt) { return from >= rows ? 0 : limit(from + cnt - 1 < rows ? from + cnt - 1 : rows - 1); };
  const uint32_t l_min = limit(r0), l_max = last_of(r0, TR), mine = last_of(wr0, 16 * NQ), mine_min = limit(wr0);

  v8 qf[NQ][KK];
  uint32_t lim[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const uint32_t r = wr0 + q * 16 + c;
    lim[q] = limit(r);
    const uint32_t i = r / G;
    const E* p = reinterpret_cast<const E*>(a.q) + (uint64_t)(first + i) * a.q_token + (uint64_t)(h * G + (r - i * G)) * a.q_head;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      const uint32_t d = g * (DP / 4) + k * 8;
      qf[q][k] = flipped<E>(load_q8<E>(p + d, r < rows && d < D, a.q_vec), a.flip);
    }
  }
  const uint32_t share = 64 * ((l_max + a.splits * 64 - 1) / (a.splits * 64));
  const uint64_t k0_64 = (uint64_t)split * share;
  const uint32_t k0 = k0_64 < l_max ? (uint32_t)k0_64 : l_max, k1 = share < l_max - k0 ? k0 + share : l_max;
  Rows<NQ, VJ> st;
  clear(st, lim, k0);
  const int32_t* table = a.s.table + b * a.s.table_stride;
  const uint32_t head_off = h * T * D;
  uint32_t k_lane[KW / 4], v_lane[4];   // this lane's bytes of a tile, as in fl_kv_attend
#pragma unroll
  for (int i = 0; i < KW / 4; ++i) k_lane[i] = c * D + (g * (DP / 4) + 16 * i < D ? g * (DP / 4) + 16 * i : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) v_lane[i] = (4 * g + i) * D + ((uint32_t)(c * VJ) < D ? c * VJ : 0);
  uint32_t bad = 0, nan_steps = 0, left_out = 0;

  // this wavefront's tile of the 64 keys from k on: where it lies, its codes, its operands
  struct Where { uint32_t pos, page, off; bool ok; };
  const uint32_t last_tile = (k1 - 1) >> 4;            // (used when there are keys)
  const auto look_up = [&](uint32_t tv) {
    Where w;
    const uint32_t tl = tv < last_tile ? tv : last_tile, j = a.per_page == 1 ? tl : __umulhi(tl, a.per_page_inv);
    w.ok = tv <= last_tile;
    w.pos = tl << 4;
    w.off = head_off + ((tl - j * a.per_page) << 4) * D;
    w.page = (uint32_t)scalar_load(table + j);
    return w;
  };
  struct Stage { uint32_t kw[KW], vw[4][VW], pos; float ks, vs; bool ok; };
  const auto fetch = [&](Stage& s, const Where& w) {
    const bool there = w.page < a.c.n_pages;
    bad |= w.ok && !there ? 1 : 0;
    s.pos = w.pos;
    s.ok = w.ok && there;
    const uint8_t* rec = a.c.pages + (uint64_t)(there ? w.page : 0) * a.c.stride;
    const float* sc = reinterpret_cast<const float*>(rec + a.c.scales) + 2 * h;
    s.ks = scalar_load(sc);
    s.vs = scalar_load(sc + 1);
    const uint8_t *base = rec + w.off, *vb = base + a.c.side;
    asm("" : "+s"(base), "+s"(vb));
#pragma unroll
    for (int i = 0; i < KW / 4; ++i) {
      const u32x4 y = *reinterpret_cast<const u32x4*>(base + k_lane[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s.kw[4 * i + e] = y[e];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(vb + v_lane[i]);
      if constexpr (VW == 1) s.vw[i][0] = p[0];
      else if constexpr (VW == 2) { const u2 y = *reinterpret_cast<const u2*>(p); s.vw[i][0] = y[0]; s.vw[i][1] = y[1]; }
      else {
        const u32x4 y = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) s.vw[i][e] = y[e];
      }
    }
  };
  const auto stage = [&](Stage& s, bool second) {
    const int x = scale_bits(s.vs), y = scale_bits(sm_scale[wave ^ 1]);   // and of the tile that shares the step
    const bool small = s.ok && x < y && apart(x, y), take = s.ok && small == second;
    if (small) left_out = 1;
    if (!s.ok || s.pos + 16 > l_min) {   // as in fl_kv_attend: values nobody sees, and NaN, are left out
      asm volatile("");
      uint32_t seen = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool keep = s.ok && s.pos + 4 * g + i < l_max;
#pragma unroll
        for (int e = 0; e < VW; ++e) s.vw[i][e] = without_nan(keep ? s.vw[i][e] : 0, seen);
      }
      if (__ballot(seen != 0)) nan_steps = 1;
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) sm_k[(wave * KK + kk) * 64 + lane] = codes8<E>(s.kw[2 * kk], s.kw[2 * kk + 1]);
#pragma unroll
    for (int e = 0; e < VW; ++e) {
      h2 v[2][4];
      interleave(s.vw[0][e], s.vw[1][e], v[0]);
      interleave(s.vw[2][e], s.vw[3][e], v[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u2* at = reinterpret_cast<u2*>(&sm_v[((wave >> 1) * VJ + 4 * e + j) * 64 + lane]) + (wave & 1);
        *at = u2{__builtin_bit_cast(uint32_t, v[0][j]), __builtin_bit_cast(uint32_t, v[1][j])};
      }
    }
    if (lane == 0) sm_tile[wave] = f4{fmaxf(s.ok ? s.ks * a.scale2 : 0.f, kLeast), take ? s.vs : 0.f, take ? 1.f : 0.f, 0.f};
  };

  if (threadIdx.x == 0) sm_nan = sm_left_out = 0;
  for (bool second = false; k0 < k1; second = true) {   // all tiles but the small ones beside large ones; then those, if there are any
    Stage s;
    Where w = look_up((k0 >> 4) + wave);
    fetch(s, w);
    w = look_up((k0 >> 4) + 4 + wave);
    for (uint32_t k = k0; k < k1; k += 64) {
      if (lane == 0) sm_scale[wave] = s.ok ? s.vs : 0.f;
      __syncthreads();                                 // the last 64 keys have been used
      stage(s, second);
      fetch(s, w);
      w = look_up((k >> 4) + 8 + wave);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t p0 = k + 32 * u;
        if (p0 >= mine || p0 >= k1) break;
        const f4 t0 = sm_tile[2 * u], t1 = sm_tile[2 * u + 1];
        f4 sc[NQ][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int q = 0; q < NQ; ++q) sc[q][t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            const v8 kf = sm_k[((2 * u + t) * KK + kk) * 64 + lane];
#pragma unroll
            for (int q = 0; q < NQ; ++q) sc[q][t] = Frag<E>::mfma(kf, qf[q][kk], sc[q][t]);
          }
        }
        if (p0 + 32 > mine_min || __ballot(t0[2] * t1[2] == 0.f)) {
          asm volatile("");
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int q = 0; q < NQ; ++q)
                if (!((t ? t1 : t0)[2] != 0.f && p0 + 16 * t + 4 * g + i < lim[q])) sc[q][t][i] = -kInf;
        }
        h8 pf[NQ];
        soften(st, sc, t0[0], t1[0], t0[1], t1[1], pf);
#pragma unroll
        for (int j = 0; j < VJ; ++j) {
          const h8 vf = sm_v[(u * VJ + j) * 64 + lane];
#pragma unroll
          for (int q = 0; q < NQ; ++q) st.o[q][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[q], st.o[q][j], 0, 0, 0);
        }
      }
    }
    if (left_out) sm_left_out = 1;
    __syncthreads();
    if (second || !sm_left_out) break;
  }
  if (nan_steps) sm_nan = 1;
  __syncthreads();
  if (sm_nan) {   // a NaN value that not every row of the workgroup sees: into the sums of those that do
    for (uint32_t tv = k0 >> 4; tv << 4 < k1; ++tv) {
      const Where w = look_up(tv);
      const bool ok = w.page < a.c.n_pages;
      if (!ok || w.pos + 16 <= l_min) continue;
      const uint8_t* base = a.c.pages + (uint64_t)w.page * a.c.stride + a.c.side + w.off;
      for (uint32_t kx = 0; kx < 16 && w.pos + kx < l_max; ++kx)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < VJ; ++j) {
            const uint32_t d = (4 * g + i) * VJ + j;
            const bool nan = d < D && (base[kx * D + d] & 0x7f) == 0x7f;
#pragma unroll
            for (int q = 0; q < NQ; ++q) st.o[q][j][i] += nan && w.pos + kx < lim[q] ? kNan : 0.f;
          }
    }
  }
  if (bad && lane == 0) report(a.s.status);
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const uint32_t r = wr0 + q * 16 + c;
    const float l = column_sum(st.l[q]), f = l == 0.f ? 0.f : 1.f / l;   // (then the scale: together they may leave the range)
    if (r >= rows) continue;
    float v[4 * VJ];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VJ; ++j) v[i * VJ + j] = __builtin_amdgcn_ldexpf(st.o[q][j][i] * f, st.ev - 127);
#pragma unroll
    for (int u = 0; u < 4 * VJ; u += 8) emit8<E>(a, split, first, h, r, l == 0.f ? -kInf : st.ref[q], l, v + u, g * 4 * VJ + u, g == 0 && u == 0);
  }
}

// The splits' results of every row, weighted by what their shares of the keys add up to.  Rows are numbered as in
// fl_kv_attend, so those of no sequence are not touched.  A wavefront joins one row: with DL = D / 4 lanes to a split it
// reads 64 / DL splits at a time, eight such loads under way.  What it takes is the start of a launch and one or two trips to
// memory (5 us for few splits).
constexpr uint32_t kMostSplits = 256;
template <class E, bool SEL>
__global__ __launch_bounds__(256) void fl_kv_join(const AttendArgs a, uint32_t TR) {
  warm_kernel_args(a);
  const uint32_t H = a.c.H, G = a.G, D = a.c.D, lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const uint32_t h = blockIdx.x % H, x = blockIdx.x / H;
  uint32_t tile, r0, rows, tok0 = 0;
  Item it;
  if constexpr (SEL) {
    const uint32_t per = (G + TR - 1) / TR, t = x / per;
    if (!find_item(a.s, a.c.T, t, [](uint32_t m, uint32_t) { return m; }, it)) return;
    tok0 = it.local;
    tile = x - t * per;
  } else {
    if (!find_item(a.s, a.c.T, x, [&](uint32_t m, uint32_t) { return (m * G + TR - 1) / TR; }, it)) return;
    tile = it.local;
  }
  const uint32_t first = it.first, n = it.n;
  if constexpr (SEL) { r0 = tok0 * G + tile * TR; rows = (tok0 + 1) * G; } else { r0 = tile * TR; rows = n * G; }
  const uint64_t row_out = (uint64_t)a.s.n_tokens * H * G;
  const uint32_t r = r0 + blockIdx.y * 4 + wave;
  if (r >= rows) return;
  const uint32_t i = r / G;
  const uint64_t tok = first + i, hq = h * G + (r - i * G), at = tok * H * G + hq;
  const uint32_t DL = D <= 64 ? 16 : D <= 128 ? 32 : 64, SP = 64 / DL, d = (lane & (DL - 1)) * 4, sub = lane / DL;

  float part[kMostSplits / 64], top = -kInf;
#pragma unroll
  for (uint32_t k = 0; k < kMostSplits / 64; ++k) {
    const uint32_t s = 64 * k + lane;
    part[k] = -kInf;
    if (64 * k < a.splits) part[k] = s < a.splits ? a.part_l[s * row_out + at] : -kInf;
    top = fmaxf(top, part[k]);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float base = top == -kInf ? 0.f : top;
  float sum = 0.f;
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  const float* mine = a.part_o + at * D + (d < D ? d : 0);
  const uint64_t step = row_out * D;
#pragma unroll
  for (uint32_t k = 0; k < kMostSplits / 64; ++k) {
    if (64 * k >= a.splits) break;
    const float w = part[k] == -kInf ? 0.f : exp2_fast(part[k] - base) * (1.f / kMostSplits);   // (no sum of them passes what it averages)
    sum += w;
    const uint32_t cnt = a.splits - 64 * k < 64 ? a.splits - 64 * k : 64;
    // A share of no keys has a weight of 0 and may have written no row: what is read for it is not used.
    const auto add = [&](auto many, uint32_t s) {
      constexpr uint32_t U = decltype(many)::value;
      f4 o[U];
      float ws[U];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t m = s + u * SP + sub;
        ws[u] = __shfl(w, (int)(m < cnt ? m : cnt - 1));
        ws[u] = m < cnt ? ws[u] : 0.f;
        o[u] = *reinterpret_cast<const f4*>(mine + (64 * k + (m < cnt ? m : cnt - 1)) * step);
      }
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += ws[u] == 0.f ? 0.f : o[u][e] * ws[u];
    };
    if (cnt <= 2 * SP) add(std::integral_constant<uint32_t, 2>{}, 0);
    else
      for (uint32_t s = 0; s < cnt; s += 8 * SP) add(std::integral_constant<uint32_t, 8>{}, s);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    for (uint32_t o = DL; o < 64; o <<= 1) acc[e] += __shfl_xor(acc[e], (int)o);
  const float f = sum == 0.f ? 0.f : 1.f / sum, lg = sum == 0.f ? -kInf : base + __builtin_amdgcn_logf(sum * kMostSplits);
  if (lane == 0) {
    if (a.lse) a.lse[at] = lg * 0.6931471805599453f;
    if (a.lse2) a.lse2[at] = lg;
  }
  if (sub == 0 && d < D) {
    E* p = reinterpret_cast<E*>(a.out) + tok * a.o_token + hq * a.o_head + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = (E)(acc[e] * f);
  }
}

// What every key of a sequence was worth to the call's queries: the probabilities exp2(s - lse) summed over the rows of
// its key-value head, on top of w_in.  A wavefront owns NT tiles of 16 keys at a time and walks over all rows, so the
// sums need no atomics; the next tiles' codes are on their way meanwhile.  Rows that fit one tile are loaded once.
// Memory bounds it: 16 sequences of up to 8192 tokens, 8 heads of 128 channels, 88 MB of keys in 26 us, 3.4 TB/s.
template <class E, int DP>
__global__ __launch_bounds__(256) void fl_kv_weights(const AttendArgs a) {
  warm_kernel_args(a);
  constexpr int KK = DP / 32, KW = DP / 16, NT = 2;
  typedef typename Frag<E>::v8 v8;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const uint32_t H = a.c.H, G = a.G, T = a.c.T, D = a.c.D, h = blockIdx.y, b = blockIdx.z;
  const uint32_t wave = blockIdx.x * 4 + uniform(threadIdx.x >> 6), step = gridDim.x * 4 * NT;   // in tiles
  uint32_t first, n;
  uniform_tokens(a.s, b, first, n);
  const uint32_t len = uniform_len(a.s, T, b), rows = n * G, tiles = rows ? (len + 15) >> 4 : 0, last_tile = tiles - 1, span = (a.w_width + 15) >> 4;
  const float* w_in = a.w_in ? a.w_in + b * a.wi_seq + h * a.wi_head : nullptr;
  float* w_out = a.w_out + b * a.wo_seq + h * a.wo_head;
  if (len > a.w_width && lane == 0) report(a.s.status);
  const int32_t* table = a.s.table + b * a.s.table_stride;
  uint32_t k_lane[KW / 4], bad = 0;
#pragma unroll
  for (int i = 0; i < KW / 4; ++i) k_lane[i] = c * D + (g * (DP / 4) + 16 * i < D ? g * (DP / 4) + 16 * i : 0);

  struct Stage { uint32_t kw[NT][KW]; float kc[NT]; bool ok[NT]; };
  const auto fetch = [&](Stage& s, uint32_t t0) {     // (past the end: the last tile again)
    uint32_t page[NT], slot[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t tl = t0 + t < tiles ? t0 + t : last_tile, j = a.per_page == 1 ? tl : __umulhi(tl, a.per_page_inv);
      slot[t] = (tl - j * a.per_page) << 4;
      page[t] = (uint32_t)scalar_load(table + j);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const bool there = page[t] < a.c.n_pages;
      s.ok[t] = t0 + t < tiles && there;
      bad |= there ? 0 : 1;
      const uint8_t* rec = a.c.pages + (uint64_t)(there ? page[t] : 0) * a.c.stride;
      s.kc[t] = fmaxf(scalar_load(reinterpret_cast<const float*>(rec + a.c.scales) + 2 * h) * a.scale2, kLeast);
      const uint8_t* base = rec + (uint64_t)(h * T + slot[t]) * D;
      asm("" : "+s"(base));
#pragma unroll
      for (int i = 0; i < KW / 4; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(base + k_lane[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s.kw[t][4 * i + e] = w[e];
      }
    }
  };
  v8 qf[KK];
  float lg = 0.f;
  uint32_t lim = 0;
  const auto load_rows = [&](uint32_t r0) {
    const uint32_t r = r0 + c, i = r / G;
    const bool in = r < rows;
    const uint64_t tok = first + i, hq = h * G + (r - i * G);
    const E* p = reinterpret_cast<const E*>(a.q) + tok * a.q_token + hq * a.q_head;
#pragma unroll
    for (int k = 0; k < KK; ++k) qf[k] = flipped<E>(load_q8<E>(p + g * (DP / 4) + k * 8, in && g * (DP / 4) + k * 8 < D, a.q_vec), a.flip);
    lg = in ? a.lse2[tok * H * G + hq] : 0.f;
    lg = lg == -kInf ? kInf : lg;                     // no key is worth anything to such a row
    const int64_t l = !in ? 0 : a.causal ? (int64_t)len - n + i + 1 : len;
    lim = l > 0 ? (uint32_t)l : 0;
  };
  const auto work = [&](const Stage& s, uint32_t t0) {
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    if (t0 < tiles) {
      for (uint32_t r0 = 0; r0 < rows; r0 += 16) {
        if (rows > 16) load_rows(r0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < KK; ++k) x = Frag<E>::mfma(codes8<E>(s.kw[t][2 * k], s.kw[t][2 * k + 1]), qf[k], x);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = exp2_fast(__builtin_fmaf(x[e], s.kc[t], -lg));
            acc[t][e] += s.ok[t] && ((t0 + t) << 4) + 4 * g + e < lim ? p : 0.f;
          }
        }
      }
    }
    // lane c of group g writes position 4 g + (c & 3) of tile c >> 2
    float mine = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = acc[t][e];
        v += __uint_as_float(dpp_u32<0xb1>(__float_as_uint(v)));    // quad_perm 1 0 3 2
        v += __uint_as_float(dpp_u32<0x4e>(__float_as_uint(v)));    // quad_perm 2 3 0 1
        v += __uint_as_float(dpp_u32<0x141>(__float_as_uint(v)));   // mirrored in 8
        v += __uint_as_float(dpp_u32<0x140>(__float_as_uint(v)));   // mirrored in 16
        mine = c == 4 * t + e ? v : mine;
      }
    const uint32_t p = (t0 << 4) + 16 * (c >> 2) + 4 * g + (c & 3);
    if (c < 4 * NT && p < a.w_width && (p < len || w_in != w_out)) w_out[p] = (w_in ? w_in[p] : 0.f) + (p < len ? mine : 0.f);
  };

  const uint32_t end = tiles > span ? tiles : span;
  uint32_t t0 = wave * NT;
  if (t0 >= end) return;
  Stage now, next;
  if (tiles) {
    fetch(now, t0);
    load_rows(0);
  }
  for (; t0 < end; t0 += step) {
    if (tiles) fetch(next, t0 + step);
    work(now, t0);
    now = next;
  }
  if (bad && lane == 0) report(a.s.status);
}

// ------------------------------------------------------------------------------------------------
// the choice of pages, and of tokens
// ------------------------------------------------------------------------------------------------
struct SelectArgs {
  Cache c;
  Seqs s;
  const void* q;
  uint64_t q_token, q_head;
  uint32_t G, causal, q_vec, first, last, count, parts, heads_wg;
  float* scores;              // [n_tokens][H][width]
  int32_t* out;               // [n_tokens][H][count]
};

__device__ __forceinline__ uint32_t token_limit(const SelectArgs& a, uint32_t len, uint32_t n, uint32_t i) {
  if (!a.causal) return len;
  const int64_t l = (int64_t)len - n + i + 1;
  return l > 0 ? (uint32_t)l : 0;
}

// score(page) = max over the group's heads of ks * qs * sum_d q8_d (q8_d > 0 ? high_d : low_d): an estimate of the
// largest product that a key of the page can have with the query, in whole numbers (8-bit queries against the page's
// 8-bit bounds), so equal scores are equal and the choice does not depend on the order of a sum.  The sum splits into
// max(q8, 0) . high - max(-q8, 0) . low, two runs of 16 x 16 x 64 integer matrix instructions whose operands are the
// bytes of the record as they lie.  Memory bounds it: bounds of 2 KiB in records of 34 KiB, 65536 pages of 8 heads of 128
// channels, 139 MB in 36 us, 3.8 TB/s; up to 2048 pages for each of 16 tokens, 42 MB, take 18.
template <class E, int DP>
__global__ __launch_bounds__(512) void fl_kv_score(const SelectArgs a) {
  warm_kernel_args(a);
  constexpr int KK = DP / 64;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const uint32_t wave = uniform(threadIdx.x >> 6), H = a.c.H, G = a.G, T = a.c.T, D = a.c.D, HW = a.heads_wg, groups = (H + HW - 1) / HW;
  const uint32_t h = blockIdx.x % groups * HW + wave % HW, part = blockIdx.x / groups;
  if (h >= H) return;
  Item it;
  if (!find_item(a.s, T, blockIdx.y, [](uint32_t m, uint32_t) { return m; }, it)) return;
  const uint32_t b = it.b, i = it.local, first = it.first, n = it.n, lim = token_limit(a, it.len, n, i), pages = (lim + T - 1) / T;
  const uint32_t subs = (blockDim.x >> 6) / HW, step = a.parts * subs * 32;   // 32 pages to a wavefront at a time
  uint32_t p0 = (part * subs + wave / HW) * 32;
  if (p0 >= pages) return;
  const uint64_t tok = first + i;
  const int32_t* table = a.s.table + b * a.s.table_stride;
  float* out = a.scores + (tok * H + h) * a.s.width;

  struct Bounds { i4 lo[2][KK], hi[2][KK]; float ks[2]; };
  uint32_t d_lane[KK];   // dims beyond D meet zeros of the query
#pragma unroll
  for (int k = 0; k < KK; ++k) d_lane[k] = k * 64 + g * 16 < D ? k * 64 + g * 16 : 0;
  uint32_t bad = 0;
  const auto number = [&](uint32_t p, int32_t* pg) {       // page numbers of rows c of the two tiles
#pragma unroll
    for (int t = 0; t < 2; ++t) pg[t] = table[p + 16 * t + c < pages ? p + 16 * t + c : pages - 1];
  };
  const auto fetch = [&](const int32_t* pg, Bounds& x) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool there = (uint32_t)pg[t] < a.c.n_pages;
      bad |= there ? 0 : 1;
      const uint8_t* rec = a.c.pages + (uint64_t)(there ? (uint32_t)pg[t] : 0) * a.c.stride;
      const uint8_t *lo = rec + a.c.low + h * D, *hi = rec + a.c.high + h * D;
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        x.hi[t][k] = *reinterpret_cast<const i4*>(hi + d_lane[k]);
        x.lo[t][k] = *reinterpret_cast<const i4*>(lo + d_lane[k]);
      }
      x.ks[t] = *(reinterpret_cast<const float*>(rec + a.c.scales) + 2 * h);
      if (!there) x.ks[t] = kNan;
    }
  };
  int32_t pg[2], later[2];
  number(p0, pg);
  number(p0 + step < pages ? p0 + step : p0, later);

  // the queries of up to 16 heads as 8-bit whole numbers, split by sign (more heads: one round for each 16)
  i4 up[KK], dn[KK];
  float scale = 0.f;
  const auto queries = [&](uint32_t h0) {
    const bool in = h0 + c < G;
    const E* q = reinterpret_cast<const E*>(a.q) + tok * a.q_token + (uint64_t)(h * G + h0 + c) * a.q_head;
    typename Frag<E>::v8 x[KK][2];
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int u = 0; u < 2; ++u) x[k][u] = load_q8<E>(q + k * 64 + g * 16 + u * 8, in && k * 64 + g * 16 < D, a.q_vec);
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = larger(amax, fabsf((float)x[k][e >> 3][e & 7]));
    bool odd = !(amax < kInf);   // (a NaN alone gives way to the numbers: it is looked for below)
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) odd |= x[k][e >> 3][e & 7] != x[k][e >> 3][e & 7];
    if (__ballot(odd)) {         // what is not finite counts as 0
      asm volatile("");
      amax = 0.f;
#pragma unroll
      for (int k = 0; k < KK; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = (float)x[k][e >> 3][e & 7];
          if (!__builtin_isfinite(v)) x[k][e >> 3][e & 7] = (E)0.f;
          else amax = larger(amax, fabsf(v));
        }
    }
    amax = column_max(amax);
    scale = 0.f;   // smallest 2^e >= amax / 127, 127 = 1.984375 * 2^6
    if (amax > 0.f) {
      const uint32_t u = __float_as_uint(amax);
      int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x7e0000u ? 6 : 5);
      if (e < -126 || u < 0x800000u) e = -126;
      scale = pow2f(e);
    }
    const float inv = inverse(scale);
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t pu = 0, pd = 0;   // positive ones, magnitudes of negative ones: the conversion to a byte cuts off below zero
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float f = (float)x[k][w >> 1][(4 * w + e) & 7];
          f = rintf(f * inv);
          pu = __builtin_amdgcn_cvt_pk_u8_f32(f, e, pu);
          pd = __builtin_amdgcn_cvt_pk_u8_f32(-f, e, pd);
        }
        up[k][w] = (int)pu;
        dn[k][w] = (int)pd;
      }
    return in;
  };

  Bounds now;
  fetch(pg, now);
  bool in = queries(0);
  for (; p0 < pages; p0 += step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) pg[t] = later[t];
    number(p0 + 2 * step < pages ? p0 + 2 * step : p0, later);
    float best[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) best[t][e] = -kInf;
    for (uint32_t h0 = 0; h0 < G; h0 += 16) {
      if (G > 16) in = queries(h0);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        i4 sum = {0, 0, 0, 0}, less = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KK; ++k) {
          sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(now.hi[t][k], up[k], sum, 0, 0, 0);
          less = __builtin_amdgcn_mfma_i32_16x16x64_i8(now.lo[t][k], dn[k], less, 0, 0, 0);
        }
        sum -= less;
#pragma unroll
        for (int e = 0; e < 4; ++e) best[t][e] = in ? fmaxf(best[t][e], (float)sum[e] * scale) : best[t][e];   // row 4 g + e: a page; column c: a head
      }
    }
    const float ks0 = now.ks[0], ks1 = now.ks[1];
    fetch(pg, now);
    float mine = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = best[t][e];
        v = larger(v, __uint_as_float(dpp_u32<0xb1>(__float_as_uint(v))));
        v = larger(v, __uint_as_float(dpp_u32<0x4e>(__float_as_uint(v))));
        v = larger(v, __uint_as_float(dpp_u32<0x141>(__float_as_uint(v))));
        v = larger(v, __uint_as_float(dpp_u32<0x140>(__float_as_uint(v))));
        v *= __shfl(t ? ks1 : ks0, 4 * g + e);
        mine = c == 4 * t + e ? (v != v ? -kInf : v) : mine;
      }
    const uint32_t p = p0 + 16 * (c >> 2) + 4 * g + (c & 3);
    if (c < 8 && p < pages) out[p] = mine;
  }
  if (bad) report(a.s.status);
}

// Numbers in their order as unsigned integers; NaN before all of them, what has to stay behind.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0;
  uint32_t u = __float_as_uint(f);
  if (u == 0x80000000u) u = 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Pick { uint32_t key, need; };
constexpr uint32_t kHeld = 16;     // keys in shared memory for each thread of a workgroup; longer rows are read again

template <int NT, bool ONE>
struct PickShared {
  uint32_t keys[ONE ? NT * kHeld : 1], hist[2048], word[4], wave[3][NT / 64];
};

// all lanes get the largest of the 64
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  uint32_t t = dpp_u32<0xb1>(v);
  v = t > v ? t : v;
  t = dpp_u32<0x4e>(v);
  v = t > v ? t : v;
  t = dpp_u32<0x141>(v);
  v = t > v ? t : v;
  t = dpp_u32<0x140>(v);
  v = t > v ? t : v;
  auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = r[0] > r[1] ? r[0] : r[1];
  r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return r[0] > r[1] ? r[0] : r[1];
}

// The k-th largest of n keys (k < n), and how many of its equals belong to the k.  2048 equal bins over the range that
// the keys span, so that keys of like size do not all count into a few; the bin that holds the k-th is taken for the
// next range until all of it belongs to the k (then the key returned is the one below it), it is one value or it holds
// no more than 64.  Keys of all
// ones (what has to be among the k) are counted apart and do not stretch the range.  The loops are short and rolled:
// with a few rows to a call, fetching straight-line code for keys in registers took longer than all else here.
template <int NT, bool ONE, class Key>
__device__ Pick kth_largest(uint32_t n, uint32_t k, Key key, PickShared<NT, ONE>& sh) {
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  uint32_t lo = 0xffffffffu, hi = 0, forced = 0;
  for (uint32_t base = tid; base < n; base += 4 * NT) {   // four loads at a time, none behind a branch
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = key(base + e * NT < n ? base + e * NT : n - 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = base + e * NT < n, all = u[e] == 0xffffffffu;
      if (ONE && in) sh.keys[base + e * NT] = u[e];
      forced += in && all ? 1 : 0;
      lo = !all && u[e] < lo ? u[e] : lo;
      hi = !all && u[e] > hi ? u[e] : hi;
    }
  }
  const auto held = [&](uint32_t i) { return ONE ? sh.keys[i] : key(i); };
  lo = ~wave_max_u32(~lo);
  hi = wave_max_u32(hi);
  forced = wave_incl_sum_u32(forced, (int)lane);
  if (lane == 63) { sh.wave[0][wave] = lo; sh.wave[1][wave] = hi; sh.wave[2][wave] = forced; }
  __syncthreads();
  {
    const uint32_t w = lane & (NT / 64 - 1);
    lo = ~wave_max_u32(~sh.wave[0][w]);
    hi = wave_max_u32(sh.wave[1][w]);
    forced = bcast_lane_u32(wave_incl_sum_u32(lane < NT / 64 ? sh.wave[2][w] : 0, (int)lane), 63);
  }
  if (forced >= k) return {0xffffffffu, k};
  k -= forced;
  for (;;) {                     // keys in [lo, hi], the k-th largest of them wanted; the range shrinks by 2048 each time
    if (lo == hi) return {lo, k};
    const int bits = 32 - __builtin_clz(hi - lo), shift = bits > 11 ? bits - 11 : 0;
    for (uint32_t i = tid; i < 2048; i += NT) sh.hist[i] = 0;
    __syncthreads();
    for (uint32_t base = tid; base < n; base += 4 * NT) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = held(base + e * NT < n ? base + e * NT : n - 1);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (base + e * NT < n && u[e] >= lo && u[e] <= hi) atomicAdd(&sh.hist[(u[e] - lo) >> shift], 1u);
    }
    __syncthreads();
    // thread t owns the OWN bins from 2047 - OWN t downwards: a scan from the top
    constexpr int OWN = 2048 / NT;
    uint32_t cnt[OWN], own = 0;
#pragma unroll
    for (int e = 0; e < OWN; ++e) { cnt[e] = sh.hist[2047 - OWN * tid - e]; own += cnt[e]; }
    const uint32_t incl = wave_incl_sum_u32(own, (int)lane);
    if (lane == 63) sh.wave[0][wave] = incl;
    __syncthreads();
    const uint32_t waves = wave_incl_sum_u32(lane < NT / 64 ? sh.wave[0][lane] : 0, (int)lane);
    uint32_t before = (wave ? bcast_lane_u32(waves, (int)wave - 1) : 0) + incl - own;
#pragma unroll
    for (int e = 0; e < OWN; ++e) {
      if (before < k && k <= before + cnt[e]) { sh.word[0] = 2047 - OWN * tid - e; sh.word[1] = k - before; sh.word[2] = 0; sh.word[3] = cnt[e]; }
      before += cnt[e];
    }
    __syncthreads();
    const uint32_t left = sh.word[3];
    lo += sh.word[0] << shift;
    hi = shift ? lo + ((1u << shift) - 1) : lo;
    k = sh.word[1];
    if (lo == hi) return {lo, k};
    if (k == left) return lo ? Pick{lo - 1, 0} : Pick{0, 0xffffffffu};   // all of the bin
    if (left <= 64) {              // collected, in any order, and compared each with each
      for (uint32_t base = tid; base < n; base += 4 * NT) {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = held(base + e * NT < n ? base + e * NT : n - 1);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (base + e * NT < n && u[e] >= lo && u[e] <= hi) sh.hist[atomicAdd(&sh.word[2], 1u)] = u[e];
      }
      __syncthreads();
      const uint32_t u = lane < left ? sh.hist[lane] : 0;
      uint32_t larger = 0, same = 0;
      for (uint32_t j = 0; j < left; ++j) {
        const uint32_t v = bcast_lane_u32(u, (int)j);
        larger += v > u ? 1 : 0;
        same += v == u ? 1 : 0;
      }
      const int l = __builtin_ctzll(__ballot(lane < left && larger < k && k <= larger + same));
      return {bcast_lane_u32(u, l), k - bcast_lane_u32(larger, l)};
    }
    __syncthreads();
  }
}

// Indices of the keys above the pick and of the first `need` equal to it, in ascending order: put(place, index, what
// `along` loads for the index).  Every wavefront looks over a run of the keys twice, for its counts and, once all counts are
// known, for its places, four times 64 at a time, so that the loads do not wait for the stores.
template <int NT, bool ONE, class Key, class Along, class Put>
__device__ void put_picked(uint32_t n, Pick pick, Key key, Along along, Put put, PickShared<NT, ONE>& sh) {
  const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), run = (n + NT - 1) / NT * 64;
  const uint32_t i0 = wave * run < n ? wave * run : n, i1 = n - i0 < run ? n : i0 + run;
  const auto held = [&](uint32_t i) { return ONE ? sh.keys[i < n ? i : n - 1] : key(i < n ? i : n - 1); };
  uint32_t above = 0, equal = 0;
  __syncthreads();
#pragma unroll 1
  for (uint32_t i = i0; i < i1; i += 64) {
    const uint32_t u = held(i + lane);
    above += (uint32_t)__popcll(__ballot(i + lane < i1 && u > pick.key));
    equal += (uint32_t)__popcll(__ballot(i + lane < i1 && u == pick.key));
  }
  if (lane == 0) { sh.wave[0][wave] = above; sh.wave[1][wave] = equal; }
  __syncthreads();
  const uint32_t sa = wave_incl_sum_u32(lane < NT / 64 ? sh.wave[0][lane] : 0, (int)lane), se = wave_incl_sum_u32(lane < NT / 64 ? sh.wave[1][lane] : 0, (int)lane);
  above = bcast_lane_u32(sa, (int)wave) - above;
  equal = bcast_lane_u32(se, (int)wave) - equal;
  const uint64_t below = (1ull << lane) - 1;
  for (uint32_t base = i0; base < i1; base += 128) {
    uint32_t u[2];
    float with[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = base + 64 * e + lane;
      with[e] = along(i < i1 ? i : i1 - 1);
      u[e] = held(i);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = base + 64 * e + lane;
      const bool in = i < i1, gt = in && u[e] > pick.key, eq = in && u[e] == pick.key;
      const uint64_t bg = __ballot(gt), be = __ballot(eq);
      const uint32_t g0 = above + (uint32_t)__popcll(bg & below), e0 = equal + (uint32_t)__popcll(be & below);
      if (gt || (eq && e0 < pick.need)) put(g0 + (e0 < pick.need ? e0 : pick.need), i, with[e]);
      above += (uint32_t)__popcll(bg);
      equal += (uint32_t)__popcll(be);
    }
  }
}

// A workgroup chooses one row's pages.  Its passes over the keys, one behind the other, bound it: 32 rows of 16384 pages
// 19 us, 128 of 2048 8 us.
template <int NT, bool ONE>
__global__ __launch_bounds__(NT) void fl_kv_pick_pages(const SelectArgs a) {
  warm_kernel_args(a);
  __shared__ PickShared<NT, ONE> sh;
  const uint32_t h = blockIdx.x % a.c.H, t = blockIdx.x / a.c.H;
  Item it;
  if (!find_item(a.s, a.c.T, t, [](uint32_t m, uint32_t) { return m; }, it)) return;
  const uint32_t lim = token_limit(a, it.len, it.n, it.local), pages = (lim + a.c.T - 1) / a.c.T;
  const uint64_t row = (uint64_t)(it.first + it.local) * a.c.H + h;
  const float* score = a.scores + row * a.s.width;
  int32_t* out = a.out + row * a.count;
  for (uint32_t k = (pages < a.count ? pages : a.count) + threadIdx.x; k < a.count; k += NT) out[k] = -1;
  if (pages <= a.count) {
    for (uint32_t k = threadIdx.x; k < pages; k += NT) out[k] = (int32_t)k;
    return;
  }
  const auto key = [&](uint32_t p) { const uint32_t u = order_key(score[p]); return p < a.first || p + a.last >= pages ? 0xffffffffu : u; };
  const Pick pick = kth_largest<NT, ONE>(pages, a.count, key, sh);
  put_picked<NT, ONE>(pages, pick, key, [](uint32_t) { return 0.f; }, [&](uint32_t at, uint32_t p, float) { out[at] = (int32_t)p; }, sh);
}

struct KeepArgs {
  Seqs s;
  uint32_t T, H, budget, first, recent, w_width, nw_width;
  const float* w;
  uint64_t w_seq, w_head, nw_seq, nw_head, kept_stride;
  float* nw;
  int32_t* kept;
  int32_t* new_lens;
};

// The same over the weights of a sequence and head: 128 rows of up to 8192 weights 17 us.
template <int NT, bool ONE>
__global__ __launch_bounds__(NT) void fl_kv_keep(const KeepArgs a) {
  warm_kernel_args(a);
  __shared__ PickShared<NT, ONE> sh;
  const uint32_t h = blockIdx.x % a.H, b = blockIdx.x / a.H;
  uint32_t len = uniform_len(a.s, a.T, b);
  if (len > a.w_width) { if (threadIdx.x == 0) report(a.s.status); len = a.w_width; }
  const float* w = a.w + b * a.w_seq + h * a.w_head;
  float* nw = a.nw + b * a.nw_seq + h * a.nw_head;
  int32_t* kept = a.kept + ((uint64_t)b * a.H + h) * a.kept_stride;
  const uint32_t m = len < a.budget ? len : a.budget;
  if (h == 0 && threadIdx.x == 0) a.new_lens[b] = (int32_t)m;
  for (uint32_t k = m + threadIdx.x; k < a.budget; k += NT) kept[k] = -1;
  for (uint32_t k = m + threadIdx.x; k < a.nw_width; k += NT) nw[k] = 0.f;
  if (len <= a.budget) {
    for (uint32_t k = threadIdx.x; k < len; k += NT) { kept[k] = (int32_t)k; nw[k] = w[k]; }
    return;
  }
  const auto key = [&](uint32_t p) { const uint32_t u = order_key(w[p]); return p < a.first || p + a.recent >= len ? 0xffffffffu : u; };
  const Pick pick = kth_largest<NT, ONE>(len, m, key, sh);
  put_picked<NT, ONE>(len, pick, key, [&](uint32_t p) { return w[p]; }, [&](uint32_t at, uint32_t p, float v) { kept[at] = (int32_t)p; nw[at] = v; }, sh);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kMaxPages = (1u << 23) - 1;   // of a sequence: positions fit 31 bits
constexpr uint32_t kMaxWidth = 0x7fffffffu;      // of a row that is written to its end: an index that strides past it must not wrap

bool aligned(const void* p, uint64_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
bool overlap(const void* a, const void* b, uint64_t bytes) { return (uintptr_t)a < (uintptr_t)b + bytes && (uintptr_t)b < (uintptr_t)a + bytes; }

int check_cache(const flh_kv_cache* k, Cache* c, const char* what) {
  if (!k->d_pages || !aligned(k->d_pages, 16)) return fl_set_error(FLH_E_ARG, "%s: the pool must be a 16-byte aligned device pointer", what);
  if (k->tokens == 0 || k->tokens % 16 || k->tokens > 256) return fl_set_error(FLH_E_ARG, "%s: %u tokens a page (a multiple of 16, up to 256)", what, k->tokens);
  if (k->dim == 0 || k->dim % 16 || k->dim > 256) return fl_set_error(FLH_E_ARG, "%s: head dim %u (a multiple of 16, up to 256)", what, k->dim);
  if (k->heads == 0 || k->heads > 1024) return fl_set_error(FLH_E_ARG, "%s: %u heads (1..1024)", what, k->heads);
  if (k->n_pages == 0 || k->n_pages > 0x7fffffffu) return fl_set_error(FLH_E_ARG, "%s: %u pages", what, k->n_pages);
  const uint64_t need = flh_kv_page_bytes(k->tokens, k->heads, k->dim);
  if (k->page_stride < need || k->page_stride % 16)
    return fl_set_error(FLH_E_ARG, "%s: page stride %llu (a multiple of 16, at least %llu)", what, (unsigned long long)k->page_stride, (unsigned long long)need);
  c->pages = (uint8_t*)k->d_pages;
  c->stride = k->page_stride;
  c->n_pages = k->n_pages;
  c->T = k->tokens;
  c->H = k->heads;
  c->D = k->dim;
  c->side = (uint64_t)c->H * c->T * c->D;
  c->low = 2 * c->side;
  c->high = c->low + (uint64_t)c->H * c->D;
  c->scales = c->high + (uint64_t)c->H * c->D;
  return FLH_OK;
}

int check_seqs(const flh_kv_seqs* k, Seqs* s, int32_t* d_status, const char* what) {
  if (!k->d_lens || !k->d_table || !d_status) return fl_set_error(FLH_E_ARG, "%s: lens, page table and status are required", what);
  if (k->n_seqs == 0 || k->n_seqs > 65535) return fl_set_error(FLH_E_ARG, "%s: %u sequences (1..65535)", what, k->n_seqs);
  if (k->table_width == 0 || k->table_stride < k->table_width || k->table_width > kMaxPages)
    return fl_set_error(FLH_E_ARG, "%s: page table of %u columns, stride %llu", what, k->table_width, (unsigned long long)k->table_stride);
  if (k->n_tokens > (1u << 24)) return fl_set_error(FLH_E_ARG, "%s: %u tokens in one call (up to 2^24)", what, k->n_tokens);
  if (!k->d_starts && k->n_tokens % k->n_seqs) return fl_set_error(FLH_E_ARG, "%s: %u tokens do not divide into %u sequences; give starts", what, k->n_tokens, k->n_seqs);
  s->starts = k->d_starts;
  s->lens = k->d_lens;
  s->table = k->d_table;
  s->table_stride = k->table_stride;
  s->width = k->table_width;
  s->n_seqs = k->n_seqs;
  s->n_tokens = k->n_tokens;
  s->per = k->d_starts ? 0 : k->n_tokens / k->n_seqs;
  s->status = d_status;
  return FLH_OK;
}

int finish(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FLH_OK : fl_set_error(FLH_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

constexpr uint64_t kMaxGroups = (1ull << 24) - 1;   // of 256 threads: a launch counts its threads in 32 bits

bool many_threads(uint32_t rows, uint32_t keys) { return keys > 256 * kHeld || (rows <= 256 && keys > 1536); }

struct Plan {
  int dp, nq, kvw;
  uint32_t tr, tiles_x, splits;
  uint64_t rows, part_o, part_l, lse2, bytes;
};

// How a call of flh_kv_attend is cut up; sizes only, so that the workspace can be asked for beforehand.
int make_plan(const flh_kv_attend_params* p, Plan* pl) {
  const uint32_t H = p->cache.heads, D = p->cache.dim, G = H ? p->q_heads / H : 0, n = p->seqs.n_tokens, B = p->seqs.n_seqs;
  if (G == 0 || p->q_heads % H) return fl_set_error(FLH_E_ARG, "flh_kv_attend: %u query heads over %u key-value heads", p->q_heads, H);
  if ((uint64_t)n * p->q_heads > 0x7fffffffull) return fl_set_error(FLH_E_ARG, "flh_kv_attend: %u tokens of %u heads", n, p->q_heads);
  pl->dp = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  const bool sel = p->d_selected != nullptr;
  const uint64_t rows = sel ? G : ((uint64_t)n * G + B - 1) / B;   // of a sequence, on average
  // Few rows, or few tiles of 128 rows: the four wavefronts of a workgroup share its keys; many: its rows, and a code is
  // converted once for 128 of them.  (8 sequences of 8192 tokens and 8 heads of 128 channels, 64, 128, 256, 512 rows to a head:
  // keys shared 49, 76, 122, 228 us, rows shared 65, 90, 132, 221; 32 such sequences, 128 and 256 rows: 244, 449 and 257,
  // 434; two, 256, 512 and 1024 rows: 43, 69, 111 and 57, 79, 122.  256 channels, 16 sequences of 4096, 32 and 128 rows: 72,
  // 233 and 176, 197.)
  const bool wide = pl->dp == 256;
  pl->kvw = sel || rows <= (wide ? 64 : 128) || (!wide && (rows + 127) / 128 * B * H <= 128) ? 4 : 1;
  pl->nq = pl->kvw == 4 && (pl->dp == 256 || rows <= 16) ? 1 : 2;
  pl->tr = 16 * pl->nq * (4 / pl->kvw);
  // workgroups that stay resident together: what their registers allow, on 256 compute units
  const uint32_t seats = 256 * (pl->kvw == 1 ? (pl->dp == 256 ? 1 : 3) : pl->dp == 256 ? 1 : pl->dp == 64 ? (pl->nq == 1 ? 5 : 3) : pl->nq == 1 ? 3 : 2);
  uint64_t tiles, est;
  if (sel) tiles = est = (uint64_t)n * ((G + pl->tr - 1) / pl->tr);
  else if (!p->seqs.d_starts) tiles = est = (uint64_t)B * (((uint64_t)(n / B) * G + pl->tr - 1) / pl->tr);
  else {
    tiles = (uint64_t)n * G / pl->tr + B;
    est = (uint64_t)n * G / pl->tr > B ? (uint64_t)n * G / pl->tr : B;
  }
  const uint64_t space = sel && p->n_selected < p->seqs.table_width ? (uint64_t)p->n_selected * p->cache.tokens : (uint64_t)p->seqs.table_width * p->cache.tokens;
  pl->splits = 1;
  const uint64_t pairs = est * H, launched = tiles * H;
  if (pl->kvw == 4 && pl->nq == 1) {
    // Up to 16 rows to a head, or 256 channels: memory bounds it, and 256 workgroups of one sequence and head each draw
    // most of what there is to be drawn.  Fewer are split until 512 run, if 1024 keys are left to each (16 sequences of
    // 131072 tokens, 8 heads: one share 1167 us, two 923, four 726), else until 256 do (one of 32768: 24 us in 32 shares,
    // 47 in 8, 29 in 96) or until no share is below 128 keys; more only if shares stay long (32 sequences of 8192: 97 us,
    // 106 in two; up to 65536: 616, 566; 48 of 16384: 300, 281).  Up to 1024 keys a join costs more than it saves (16
    // times 1024: 46 us, 47 in two).
    if (space > 1024 && pairs && pairs < 512) {
      uint64_t sp = (512 + pairs - 1) / pairs;
      if (seats < 512 || space < sp * (pairs < 256 ? 1024 : 8192)) sp = (256 + pairs - 1) / pairs;
      if (sp > seats / launched) sp = seats / launched;
      if (sp > space / 128) sp = space / 128;
      pl->splits = sp < 1 ? 1 : sp > kMostSplits ? kMostSplits : (uint32_t)sp;
    }
  } else {
    // More rows: rounds of workgroups times the longest share (in whole rounds of their wavefronts), a start and an end
    // worth some 384 keys each time, and the join, worth as much again.  (20 sequences of 8192, 64 rows: 120 us in one share, 109
    // in three, as this has it, 126 in eight; 8 of 2048: 28, 24 in four, 32 in eight.)
    const uint32_t round = pl->kvw == 4 ? 128 : 64;
    uint64_t best = ~0ull;
    const uint64_t top = pl->kvw == 4 ? kMostSplits : pairs < seats ? seats / (pairs ? pairs : 1) : 1;   // (rows shared: until the seats are taken)
    for (uint32_t sp = 1; sp <= top && (sp == 1 || (uint64_t)(sp - 1) * round < space); ++sp) {
      const uint64_t rounds = (pairs * sp + seats - 1) / seats, share = (space + (uint64_t)sp * round - 1) / ((uint64_t)sp * round) * round;
      const uint64_t cost = rounds * (share + 384) + (sp > 1 ? 384 : 0);
      if (cost < best) { best = cost; pl->splits = sp; }
    }
  }
  if (tiles * H * pl->splits > kMaxGroups) return fl_set_error(FLH_E_ARG, "flh_kv_attend: too much for one launch");
  pl->tiles_x = (uint32_t)tiles;
  pl->rows = (uint64_t)n * p->q_heads;
  uint64_t at = 0;
  pl->part_o = at;
  if (pl->splits > 1) at += pl->splits * pl->rows * D * 4;
  pl->part_l = at;
  if (pl->splits > 1) at += pl->splits * pl->rows * 4;
  pl->lse2 = at;
  if (p->d_weights) at += pl->rows * 4;
  pl->bytes = at;
  return FLH_OK;
}

template <class E, int DP, int NQ>
void launch_attend(const AttendArgs& a, const Plan& pl, hipStream_t st) {
  const dim3 grid(a.tiles_x * a.c.H * a.splits);
  if (pl.kvw == 1) FL_LAUNCH((fl_kv_attend_rows<E, DP>), grid, dim3(256), 0, st, a);
  else if (a.sel) FL_LAUNCH((fl_kv_attend<E, DP, NQ, true>), grid, dim3(256), 0, st, a);
  else FL_LAUNCH((fl_kv_attend<E, DP, NQ, false>), grid, dim3(256), 0, st, a);
}

template <class E>
void run_attend(const AttendArgs& a, const Plan& pl, hipStream_t st) {
  if (a.tiles_x) {
    if (pl.dp == 64) {
      if (pl.nq == 1) launch_attend<E, 64, 1>(a, pl, st);
      else launch_attend<E, 64, 2>(a, pl, st);
    } else if (pl.dp == 128) {
      if (pl.nq == 1) launch_attend<E, 128, 1>(a, pl, st);
      else launch_attend<E, 128, 2>(a, pl, st);
    } else {
      launch_attend<E, 256, 1>(a, pl, st);
    }
  }
  if (pl.splits > 1 && a.tiles_x) {
    const dim3 grid(a.tiles_x * a.c.H, pl.tr / 4);
    if (a.sel) FL_LAUNCH((fl_kv_join<E, true>), grid, dim3(256), 0, st, a, pl.tr);
    else FL_LAUNCH((fl_kv_join<E, false>), grid, dim3(256), 0, st, a, pl.tr);
  }
  if (a.w_out) {
    // as many workgroups as stay resident, or what there is to do
    const uint64_t span = (uint64_t)a.s.width * a.c.T > a.w_width ? (uint64_t)a.s.width * a.c.T : a.w_width, rows = (uint64_t)a.s.n_seqs * a.c.H;
    const uint64_t most = (span + 127) / 128, want = (1024 + rows - 1) / rows;
    const dim3 grid((uint32_t)(want < most ? want : most), a.c.H, a.s.n_seqs);
    if (pl.dp == 64) FL_LAUNCH((fl_kv_weights<E, 64>), grid, dim3(256), 0, st, a);
    else if (pl.dp == 128) FL_LAUNCH((fl_kv_weights<E, 128>), grid, dim3(256), 0, st, a);
    else FL_LAUNCH((fl_kv_weights<E, 256>), grid, dim3(256), 0, st, a);
  }
}

// As many wavefronts to a head of a page as keep its rows in registers, 8 of them a lane at most.  (One wavefront that
// reads longer blocks twice, four rows at a time, against four: 29 sequences of 1634 tokens, 12 heads of 256 channels,
// evicted into pages of 32 tokens 235 us, 123; 33 of up to 4140, 8 heads of 128, stored in pages of 64 146 us, 117; against
// sixteen, pages of 256 193 us, 147.  Eight wavefronts with four rows a lane each in place of four with eight: the same.)
template <class E, bool EVICT>
void launch_pack(const PackArgs& a, uint32_t items, hipStream_t st) {
  const uint32_t rp = 64 / (a.c.D / 8), rows = (a.c.T + rp - 1) / rp;   // 128 at most
  const dim3 heads4(items, (a.c.H + 3) / 4), heads(items, a.c.H);
  if (rows <= 4) FL_LAUNCH((fl_kv_pack<E, EVICT, 4, 1>), heads4, dim3(256), 0, st, a);
  else if (rows <= 8) FL_LAUNCH((fl_kv_pack<E, EVICT, 8, 1>), heads4, dim3(256), 0, st, a);
  else if (rows <= 16) FL_LAUNCH((fl_kv_pack<E, EVICT, 4, 4>), heads, dim3(256), 0, st, a);
  else if (rows <= 32) FL_LAUNCH((fl_kv_pack<E, EVICT, 8, 4>), heads, dim3(256), 0, st, a);
  else if (rows <= 64) FL_LAUNCH((fl_kv_pack<E, EVICT, 4, 16>), heads, dim3(1024), 0, st, a);
  else FL_LAUNCH((fl_kv_pack<E, EVICT, 8, 16>), heads, dim3(1024), 0, st, a);
}

}  // namespace

extern "C" {

uint64_t flh_kv_page_bytes(uint32_t tokens, uint32_t heads, uint32_t dim) {
  return (2ull * heads * tokens * dim + 2ull * heads * dim + 8ull * heads + 127) / 128 * 128;
}

int flh_kv_store(const flh_kv_store_params* p, void* stream) {
  if (!p) return fl_set_error(FLH_E_ARG, "flh_kv_store: null parameters");
  PackArgs a;
  memset(&a, 0, sizeof(a));
  int rc = check_cache(&p->cache, &a.c, "flh_kv_store");
  if (!rc) rc = check_seqs(&p->seqs, &a.s, p->d_status, "flh_kv_store");
  if (rc) return rc;
  if (p->type > FLH_KV_FP32) return fl_set_error(FLH_E_ARG, "flh_kv_store: type %u", p->type);
  const uint32_t esz = p->type == FLH_KV_FP32 ? 4 : 2;
  if (p->seqs.n_tokens && (!p->d_k || !p->d_v || !aligned(p->d_k, esz) || !aligned(p->d_v, esz))) return fl_set_error(FLH_E_ARG, "flh_kv_store: keys and values are required");
  if (p->seqs.n_tokens == 0) return FLH_OK;
  if ((rc = fl_need_init())) return rc;
  a.src[0] = p->d_k;
  a.src[1] = p->d_v;
  a.token_stride[0] = p->k_token_stride;
  a.token_stride[1] = p->v_token_stride;
  a.head_stride[0] = p->k_head_stride;
  a.head_stride[1] = p->v_head_stride;
  const uint64_t unit = 16 / esz, strides = p->k_token_stride | p->v_token_stride | p->k_head_stride | p->v_head_stride;
  a.vec = aligned(p->d_k, 16) && aligned(p->d_v, 16) && strides % unit == 0;
  // a sequence's new tokens touch at most n / T + 2 pages
  const uint32_t items = a.s.n_tokens / a.c.T + 2 * a.s.n_seqs;
  fl_prof().kid = 8;
  const hipStream_t st = (hipStream_t)stream;
  if (p->type == FLH_KV_BF16) launch_pack<__bf16, false>(a, items, st);
  else if (p->type == FLH_KV_FP16) launch_pack<_Float16, false>(a, items, st);
  else launch_pack<float, false>(a, items, st);
  return finish("flh_kv_store");
}

int64_t flh_kv_attend_workspace_bytes(const flh_kv_attend_params* p) {
  Plan pl;
  if (!p) return fl_set_error(FLH_E_ARG, "flh_kv_attend_workspace_bytes: null parameters");
  if (!p->seqs.n_seqs || !p->cache.tokens) return fl_set_error(FLH_E_ARG, "flh_kv_attend_workspace_bytes: no sequences or no page size");
  const int rc = make_plan(p, &pl);
  return rc ? rc : (int64_t)pl.bytes;
}

int flh_kv_attend(const flh_kv_attend_params* p, void* stream) {
  if (!p) return fl_set_error(FLH_E_ARG, "flh_kv_attend: null parameters");
  AttendArgs a;
  memset(&a, 0, sizeof(a));
  int rc = check_cache(&p->cache, &a.c, "flh_kv_attend");
  if (!rc) rc = check_seqs(&p->seqs, &a.s, p->d_status, "flh_kv_attend");
  if (rc) return rc;
  if (p->type != FLH_KV_BF16 && p->type != FLH_KV_FP16) return fl_set_error(FLH_E_ARG, "flh_kv_attend: type %u (bf16 or fp16)", p->type);
  if (p->seqs.n_tokens && (!p->d_q || !p->d_out || !aligned(p->d_q, 2) || !aligned(p->d_out, 2))) return fl_set_error(FLH_E_ARG, "flh_kv_attend: queries and output are required");
  if (!(fabsf(p->scale) * 1.4426950408889634f < kInf)) return fl_set_error(FLH_E_ARG, "flh_kv_attend: a scale of %g", (double)p->scale);
  if (p->d_selected && (p->n_selected == 0 || p->n_selected > kMaxPages)) return fl_set_error(FLH_E_ARG, "flh_kv_attend: %u selected pages", p->n_selected);
  if (p->d_selected && p->d_weights) return fl_set_error(FLH_E_ARG, "flh_kv_attend: weights are kept over all pages, not over selected ones");
  if (!p->d_weights && p->d_weights_in) return fl_set_error(FLH_E_ARG, "flh_kv_attend: weights to start from, but none to write");
  if (p->d_weights && (p->weights_width == 0 || p->weights_width > kMaxWidth)) return fl_set_error(FLH_E_ARG, "flh_kv_attend: weights of %u positions (1..2^31 - 1)", p->weights_width);
  Plan pl;
  if ((rc = make_plan(p, &pl))) return rc;
  if (pl.bytes && (!p->d_workspace || !aligned(p->d_workspace, 16) || p->workspace_bytes < pl.bytes))
    return fl_set_error(FLH_E_ARG, "flh_kv_attend: a workspace of %llu bytes is needed", (unsigned long long)pl.bytes);
  if (p->seqs.n_tokens == 0 && !p->d_weights) return FLH_OK;
  if ((rc = fl_need_init())) return rc;
  a.q = p->d_q;
  a.out = p->d_out;
  a.lse = p->d_lse;
  a.q_token = p->q_token_stride;
  a.q_head = p->q_head_stride;
  a.o_token = p->out_token_stride;
  a.o_head = p->out_head_stride;
  a.G = p->q_heads / p->cache.heads;
  a.tiles_x = pl.tiles_x;
  a.splits = pl.splits;
  a.per_page = a.c.T / 16;
  a.per_page_inv = 0xffffffffu / a.per_page + 1;   // (one tile a page: not used)
  a.scale2 = fabsf(p->scale) * 1.4426950408889634f;
  a.flip = p->scale < 0.f ? 0x80008000u : 0u;
  a.causal = p->causal != 0;
  a.q_vec = aligned(p->d_q, 16) && (p->q_token_stride | p->q_head_stride) % 8 == 0;
  a.o_vec = aligned(p->d_out, 16) && (p->out_token_stride | p->out_head_stride) % 8 == 0;
  a.sel = p->d_selected;
  a.count = p->n_selected;
  uint8_t* ws = (uint8_t*)p->d_workspace;
  a.part_o = (float*)(ws + pl.part_o);
  a.part_l = (float*)(ws + pl.part_l);
  a.lse2 = p->d_weights ? (float*)(ws + pl.lse2) : nullptr;
  a.w_in = p->d_weights_in;
  a.w_out = p->d_weights;
  a.wi_seq = p->weights_in_seq_stride;
  a.wi_head = p->weights_in_head_stride;
  a.wo_seq = p->weights_seq_stride;
  a.wo_head = p->weights_head_stride;
  a.w_width = p->weights_width;
  fl_prof().kid = 9;
  const hipStream_t st = (hipStream_t)stream;
  if (p->seqs.n_tokens == 0) a.tiles_x = 0;
  if (p->type == FLH_KV_BF16) run_attend<__bf16>(a, pl, st);
  else run_attend<_Float16>(a, pl, st);
  return finish("flh_kv_attend");
}

uint64_t flh_kv_select_workspace_bytes(uint32_t n_tokens, uint32_t heads, uint32_t table_width) { return 4ull * n_tokens * heads * table_width; }

int flh_kv_select(const flh_kv_select_params* p, void* stream) {
  if (!p) return fl_set_error(FLH_E_ARG, "flh_kv_select: null parameters");
  SelectArgs a;
  memset(&a, 0, sizeof(a));
  int rc = check_cache(&p->cache, &a.c, "flh_kv_select");
  if (!rc) rc = check_seqs(&p->seqs, &a.s, p->d_status, "flh_kv_select");
  if (rc) return rc;
  if (p->type != FLH_KV_BF16 && p->type != FLH_KV_FP16) return fl_set_error(FLH_E_ARG, "flh_kv_select: type %u (bf16 or fp16)", p->type);
  if (p->q_heads == 0 || p->q_heads % p->cache.heads) return fl_set_error(FLH_E_ARG, "flh_kv_select: %u query heads over %u key-value heads", p->q_heads, p->cache.heads);
  if (p->count == 0 || p->count > kMaxWidth || (uint64_t)p->first + p->last > p->count) return fl_set_error(FLH_E_ARG, "flh_kv_select: %u pages with %u first and %u last ones", p->count, p->first, p->last);
  if (p->seqs.n_tokens > 65535 || (uint64_t)p->seqs.n_tokens * p->cache.heads > kMaxGroups / 4)
    return fl_set_error(FLH_E_ARG, "flh_kv_select: %u tokens of %u heads in one call (up to 65535, and 2^22 - 1 rows)", p->seqs.n_tokens, p->cache.heads);
  if (p->seqs.n_tokens == 0) return FLH_OK;
  if (!p->d_q || !p->d_out || !aligned(p->d_q, 2)) return fl_set_error(FLH_E_ARG, "flh_kv_select: queries and output are required");
  const uint64_t need = flh_kv_select_workspace_bytes(p->seqs.n_tokens, p->cache.heads, p->seqs.table_width);
  if (!p->d_workspace || !aligned(p->d_workspace, 16) || p->workspace_bytes < need)
    return fl_set_error(FLH_E_ARG, "flh_kv_select: a workspace of %llu bytes is needed", (unsigned long long)need);
  if ((rc = fl_need_init())) return rc;
  a.q = p->d_q;
  a.q_token = p->q_token_stride;
  a.q_head = p->q_head_stride;
  a.G = p->q_heads / p->cache.heads;
  a.causal = p->causal != 0;
  a.q_vec = aligned(p->d_q, 16) && (p->q_token_stride | p->q_head_stride) % 8 == 0;
  a.first = p->first;
  a.last = p->last;
  a.count = p->count;
  a.scores = (float*)p->d_workspace;
  a.out = p->d_out;
  fl_prof().kid = 10;
  const hipStream_t st = (hipStream_t)stream;
  // The wavefronts of a workgroup take up to eight heads of the same pages: the pages' translations and the line that
  // holds their scales are then fetched by one compute unit (65536 pages of 8 heads, the same ones each time: a head to a
  // workgroup 41 us, four 31, eight 29).  2048 wavefronts over all rows (1024: 10 tokens over 7518 pages of 5 heads of 64 channels 53 us, 46 so;
  // 4096: 16 over 2048 pages of 8 heads of 128 44 us, 42 so), or 32 pages to each.
  const uint32_t waves = a.c.H >= 8 ? 8 : 4;
  a.heads_wg = a.c.H >= 8 ? 8 : a.c.H >= 4 ? 4 : a.c.H >= 2 ? 2 : 1;
  const uint32_t groups = (a.c.H + a.heads_wg - 1) / a.heads_wg;
  const uint64_t rows = (uint64_t)a.s.n_tokens * groups;
  const uint32_t per = 32 * (waves / a.heads_wg), want = (uint32_t)((2048 / waves + rows - 1) / rows), most = (a.s.width + per - 1) / per;
  a.parts = want < most ? want : most;
  const dim3 grid(a.parts * groups, a.s.n_tokens), block(64 * waves);
  const bool bf = p->type == FLH_KV_BF16;
  if (a.c.D <= 64) { if (bf) FL_LAUNCH((fl_kv_score<__bf16, 64>), grid, block, 0, st, a); else FL_LAUNCH((fl_kv_score<_Float16, 64>), grid, block, 0, st, a); }
  else if (a.c.D <= 128) { if (bf) FL_LAUNCH((fl_kv_score<__bf16, 128>), grid, block, 0, st, a); else FL_LAUNCH((fl_kv_score<_Float16, 128>), grid, block, 0, st, a); }
  else { if (bf) FL_LAUNCH((fl_kv_score<__bf16, 256>), grid, block, 0, st, a); else FL_LAUNCH((fl_kv_score<_Float16, 256>), grid, block, 0, st, a); }
  // 1024 threads to a row if there are no more rows than compute units and more than 6 keys to a thread of 256, or if 256 would
  // hold too few.  (The choice of 32 rows of 1024, 1536, 2048 and 4000 keys: 6.0, 7.4, 8.0, 11.9 us with 256 threads, 6.5, 6.8,
  // 6.8, 7.6 with 1024; 256 rows: 6.3, 7.8, 8.3, 13.4 and 7.0, 7.2, 7.2, 8.4; 512 rows: 7.0, 8.9, 9.4, 15.7 and 9.6, 9.7, 10.0, 11.3.)
  if (!many_threads(a.s.n_tokens * a.c.H, a.s.width)) FL_LAUNCH((fl_kv_pick_pages<256, true>), dim3(a.s.n_tokens * a.c.H), dim3(256), 0, st, a);
  else if (a.s.width <= 1024 * kHeld) FL_LAUNCH((fl_kv_pick_pages<1024, true>), dim3(a.s.n_tokens * a.c.H), dim3(1024), 0, st, a);
  else FL_LAUNCH((fl_kv_pick_pages<1024, false>), dim3(a.s.n_tokens * a.c.H), dim3(1024), 0, st, a);
  return finish("flh_kv_select");
}

int flh_kv_evict(const flh_kv_evict_params* p, void* stream) {
  if (!p) return fl_set_error(FLH_E_ARG, "flh_kv_evict: null parameters");
  PackArgs a;
  memset(&a, 0, sizeof(a));
  int rc = check_cache(&p->cache, &a.from, "flh_kv_evict: from");
  if (!rc) rc = check_cache(&p->to, &a.c, "flh_kv_evict: to");
  if (!rc) rc = check_seqs(&p->seqs, &a.s, p->d_status, "flh_kv_evict");
  if (rc) return rc;
  if (a.c.H != a.from.H || a.c.D != a.from.D) return fl_set_error(FLH_E_ARG, "flh_kv_evict: the caches differ in heads or head dim");
  if (!p->d_weights || !p->d_to_table || !p->d_kept || !p->d_new_weights || !p->d_new_lens) return fl_set_error(FLH_E_ARG, "flh_kv_evict: weights, tables and outputs are required");
  if (p->budget == 0 || p->budget > (1u << 30) || (uint64_t)p->first + p->recent > p->budget)
    return fl_set_error(FLH_E_ARG, "flh_kv_evict: a budget of %u with %u first and %u recent tokens", p->budget, p->first, p->recent);
  const uint32_t per = (p->budget + a.c.T - 1) / a.c.T;
  if (p->to_table_width < per || p->to_table_stride < p->to_table_width)
    return fl_set_error(FLH_E_ARG, "flh_kv_evict: %u tokens need %u pages, the new table has %u", p->budget, per, p->to_table_width);
  if (p->weights_width == 0 || p->weights_width > kMaxWidth || p->new_weights_width < p->budget || p->new_weights_width > kMaxWidth)
    return fl_set_error(FLH_E_ARG, "flh_kv_evict: weights of %u positions, new ones of %u", p->weights_width, p->new_weights_width);
  if (p->d_to_table == p->seqs.d_table && a.c.pages == a.from.pages) return fl_set_error(FLH_E_ARG, "flh_kv_evict: the new pages are those that are read");
  // (the workgroups of the other heads still read a length when the first one's writes the new one)
  if (overlap(p->d_new_lens, p->seqs.d_lens, 4ull * a.s.n_seqs)) return fl_set_error(FLH_E_ARG, "flh_kv_evict: the new lengths overlap the lengths");
  if ((uint64_t)per * a.s.n_seqs > kMaxGroups / 4 || (uint64_t)a.s.n_seqs * a.c.H > kMaxGroups / 4) return fl_set_error(FLH_E_ARG, "flh_kv_evict: too much for one launch");
  if ((rc = fl_need_init())) return rc;
  KeepArgs k;
  memset(&k, 0, sizeof(k));
  k.s = a.s;
  k.T = a.from.T;
  k.H = a.c.H;
  k.budget = p->budget;
  k.first = p->first;
  k.recent = p->recent;
  k.w_width = p->weights_width;
  k.nw_width = p->new_weights_width;
  k.w = p->d_weights;
  k.w_seq = p->weights_seq_stride;
  k.w_head = p->weights_head_stride;
  k.nw = p->d_new_weights;
  k.nw_seq = p->new_weights_seq_stride;
  k.nw_head = p->new_weights_head_stride;
  k.kept = p->d_kept;
  k.kept_stride = p->budget;
  k.new_lens = p->d_new_lens;
  a.to_table = p->d_to_table;
  a.to_stride = p->to_table_stride;
  a.kept = p->d_kept;
  a.kept_stride = p->budget;
  a.most = p->budget < p->weights_width ? p->budget : p->weights_width;
  a.per_seq = per;
  fl_prof().kid = 11;
  const hipStream_t st = (hipStream_t)stream;
  if (!many_threads(a.s.n_seqs * a.c.H, k.w_width)) FL_LAUNCH((fl_kv_keep<256, true>), dim3(a.s.n_seqs * a.c.H), dim3(256), 0, st, k);
  else if (k.w_width <= 1024 * kHeld) FL_LAUNCH((fl_kv_keep<1024, true>), dim3(a.s.n_seqs * a.c.H), dim3(1024), 0, st, k);
  else FL_LAUNCH((fl_kv_keep<1024, false>), dim3(a.s.n_seqs * a.c.H), dim3(1024), 0, st, k);
  launch_pack<__bf16, true>(a, per * a.s.n_seqs, st);
  return finish("flh_kv_evict");
}

}  // extern "C"
