// A cache in 8 bits is written and read back (the format: quantized.h).
//
// Writing follows the fused q|k|v projection: rms norm of q and k over the head (with or without weights, before or after
// the rotation), rotary embedding (adjacent or half-split pairs, over the head's leading part), position-dependent query
// scale, as attention_prep.hip has them, and k and v rounded once to codes and a scale byte a row.
#include "quantized.h"

using namespace jle;

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

// Keys are normed, turned and scaled in 64 bits (the matrix cores' rate aside, this card adds and multiplies doubles as fast as
// floats): a code is a rounding to four bits, and where the number to be rounded is itself off by float32's rounding, one code
// in some hundred thousand falls the other way.  The code is the only rounding behind that (toward_odd).  Queries, which are rounded to bfloat16, are worked on in float32, with the
// same angles.

// Sine and cosine of pos * freq in 64 bits: reduced by multiples of pi / 2 (the product and the remainder by fused
// multiply-adds with pi / 2 in two parts), then the Taylor series up to |r| <= pi / 4 (the first terms left out are
// r^17 / 17! < 5e-17 and r^18 / 18! < 3e-18).
__device__ __forceinline__ void turn_of(int pos, float freq, double& sn, double& cs) {
  constexpr double kHalfPi = 1.57079632679489661923, kHalfPiRest = 6.123233995736766e-17, kTwoOverPi = 0.63661977236758134308;
  const double a = (double)pos * (double)freq;  // (exact below position 2^29)
  const double k = rint(a * kTwoOverPi);
  const double r = fma(-k, kHalfPiRest, fma(-k, kHalfPi, a));
  const double q = r * r;
  double s = -1.0 / 1307674368000.0;  // 1 / 15!
  s = fma(s, q, 1.0 / 6227020800.0);
  s = fma(s, q, -1.0 / 39916800.0);
  s = fma(s, q, 1.0 / 362880.0);
  s = fma(s, q, -1.0 / 5040.0);
  s = fma(s, q, 1.0 / 120.0);
  s = fma(s, q, -1.0 / 6.0);
  s = fma(s * q, r, r);
  double c = 1.0 / 20922789888000.0;  // 1 / 16!
  c = fma(c, q, -1.0 / 87178291200.0);
  c = fma(c, q, 1.0 / 479001600.0);
  c = fma(c, q, -1.0 / 3628800.0);
  c = fma(c, q, 1.0 / 40320.0);
  c = fma(c, q, -1.0 / 720.0);
  c = fma(c, q, 1.0 / 24.0);
  c = fma(c, q, -0.5);
  c = fma(c, q, 1.0);
  const int quarter = (int)((long long)k & 3);
  sn = quarter == 0 ? s : quarter == 1 ? c : quarter == 2 ? -s : -c;
  cs = quarter == 0 ? c : quarter == 1 ? -s : quarter == 2 ? -c : s;
}

// A 64-bit number on its way to a code, in float32 without a rounding that the code's could follow the wrong way: its fraction
// is cut behind the 12th bit, which is set where anything but zeros goes (rounding to odd).  So the number stays on its side of
// every number of fewer bits: of the borders between codes, and of 448 times a power of two, which the scale asks for.  (Twelve,
// not the 23 of float32: a float below 2^-126 has fewer, and down to a code's smallest half step, 2^-136, it has thirteen.)
__device__ __forceinline__ float toward_odd(double y) {
  const uint64_t b = __builtin_bit_cast(uint64_t, y);
  uint32_t hi = (uint32_t)(b >> 32);
  hi = (hi & ~0xffu) | min((hi & 0xffu) | (uint32_t)b, 1u) << 8;
  return (float)__builtin_bit_cast(double, (uint64_t)hi << 32);
}

struct PrepareArgs {
  const bf16_t* qkv;
  bf16_t* q_out;
  uint8_t *codes, *scales;  // null: keys and values are not written
  const int *positions, *slots;
  const float* inv_freq;  // null: no rotation
  const float *norm_wq, *norm_wk;
  float norm_eps;  // < 0: no norm
  double per_element;  // 1 / dh
  float floor_scale, attn_scale;
  int norm_first, table_pairs, pairing, rotary_dim;  // pairing 0: (x[2j], x[2j + 1]), 1: (x[j], x[j + rotary_dim / 2])
  int N, Hq, Hkv, dh, ps;
  long long num_slots;
  Divisor key_chunks, value_quads;  // of a head: eight codes; (piece of 64 elements, element % 16)
  int* clear;  // counters of the attention behind this launch, which it starts from zero
  int num_clear;
};

constexpr int kTokens = 8;       // of a block, where there are many
constexpr int kManyTokens = 128;

template <typename F, int LPH>
__device__ __forceinline__ F over_head(F s) {
#pragma unroll
  for (int o = LPH >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  return s;
}

// 1 / sqrt(x): the hardware's estimate; in 64 bits two steps of Newton's method behind it
__device__ __forceinline__ float inverse_root(float x) { return __builtin_amdgcn_rsqf(x); }
__device__ __forceinline__ double inverse_root(double x) {
  double r = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) r = fma(0.5 * r, fma(-x * r, r, 1.0), r);
  return r;
}

// A head's numbers, eight a lane (l: the lane's place in the head), normed and turned.  F: what is computed in.  A rotation
// changes no length, so the norm's sum is that of the numbers as they come, whether the norm lies in front of the rotation or
// behind it; only its weights have a place.  turns: (cosine, sine) by pair; adjacent pairs beyond the rotated part: (1, 0).
template <typename F, int LPH, typename T2>
__device__ __forceinline__ void prepare_head(F (&x)[8], const PrepareArgs& a, const float* w, int l, bool live, const T2* turns) {
  F mul = 1;
  if (a.norm_eps >= 0.f) {
    F ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma(x[i], x[i], ss);
    mul = inverse_root(fma(over_head<F, LPH>(ss), (F)a.per_element, (F)a.norm_eps));
  }
  auto weigh = [&]() {
    const uint32_t at = live ? 8 * l : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= (F)w[at + i];
  };
  if (w != nullptr && a.norm_first) weigh();
  if (a.inv_freq != nullptr) {
    if (a.pairing == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T2 t = turns[live ? 4 * l + i : 0];
        const F p = x[2 * i], q = x[2 * i + 1], c = (F)t.x, s = (F)t.y;
        x[2 * i] = fma(p, c, -(q * s));
        x[2 * i + 1] = fma(q, c, p * s);
      }
    } else {  // (half of the rotated part is a multiple of 8: a lane's partners are all in one other lane)
      const int half = a.rotary_dim >> 1, lane = threadIdx.x & 63;
      const bool turned = 8 * l < a.rotary_dim, leading = 8 * l < half;
      const int other = turned ? (leading ? lane + half / 8 : lane - half / 8) : lane;
      const T2* mine = turns + (leading ? 8 * l : turned ? 8 * l - half : 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const F y = __shfl(x[i], other, 64);
        const T2 t = mine[i];
        x[i] = turned ? fma(x[i], (F)t.x, (leading ? -y : y) * (F)t.y) : x[i];
      }
    }
  }
  if (w != nullptr && !a.norm_first) weigh();
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= mul;
}

// LPH lanes a head (a power of two, at least dh / 8), eight neighbouring elements a lane, 64 / LPH heads of a kind (queries,
// keys, values) a wavefront at a time: a *unit*.  A block takes TB consecutive tokens and forms their sines and cosines once.
// With one token a block (few tokens) the units are shared out among gridDim.y blocks of four wavefronts and the codes go
// straight into their pages (one token of 56 heads 4.3 us, 64 of 32 5.2); with several TW wavefronts share a token, the codes
// are gathered in shared memory and written in larger pieces (8,191 tokens of 48 heads of 128: 49 us, 3.8 TB/s, 98 when every
// value was stored by itself; vector instructions bound it, 1,900 a token and wavefront): keys eight codes each, the tokens'
// side by side, values the four keys of four elements in 16 bytes where the block's tokens fill an aligned four of a page (other
// values byte by byte).
template <int LPH, int TB, int TW>
__global__ __launch_bounds__(TB > 1 ? TB * 64 * TW : 256, 4) void quantized_prepare_kernel(PrepareArgs a) {
  constexpr int HPW = 64 / LPH, THREADS = TB > 1 ? TB * 64 * TW : 256;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int l = lane & (LPH - 1), sub = lane / LPH;
  const int n0 = blockIdx.x * TB;
  const int pairs = a.table_pairs, half = a.rotary_dim >> 1;  // of a token's table; of them turned
  const int dh = a.dh, row_codes = a.Hkv * dh;
  double2* turns = reinterpret_cast<double2*>(smem);  // [TB][pairs]: for keys, and in float32 for queries
  float2* turns32 = reinterpret_cast<float2*>(turns + TB * pairs);
  uint8_t* held = reinterpret_cast<uint8_t*>(turns32 + TB * pairs);  // [2][TB][Hkv][dh], several tokens only
  __shared__ int slot_of[TB], leads[TB];
  __shared__ float temper[TB];
  __shared__ size_t code_at[TB], scales_at[TB];  // of head 0's keys: the codes of the slot's sixteen, the slot's scale byte
  if (a.num_clear > 0 && blockIdx.y == 0)
    for (int i = blockIdx.x * THREADS + threadIdx.x; i < a.num_clear; i += gridDim.x * THREADS) a.clear[i] = 0;

  const int tk = TB > 1 ? wave / TW : 0, n = n0 + tk;
  const int uq = (a.Hq + HPW - 1) / HPW, uk = a.codes != nullptr ? (a.Hkv + HPW - 1) / HPW : 0, units = uq + 2 * uk;
  const int step = TB > 1 ? TW : 4 * gridDim.y;
  const bool in_head = 8 * l < dh, token = n < a.N;
  constexpr int AHEAD = TB > 1 ? 4 : 1;  // units' rows asked for at once
  u32x4 raw[AHEAD], next[AHEAD];
  const uint32_t in_unit = sub * dh + 8 * l;  // a lane's first element among a unit's
  const bf16_t* row = a.qkv + (size_t)(token ? n : 0) * (a.Hq + 2 * a.Hkv) * dh;
  // a unit's kind, its first head and, of those, how many there are
  auto unit = [&](int u, int& kind, int& h0) {
    kind = u < uq ? 0 : u < uq + uk ? 1 : 2;
    h0 = (kind == 0 ? u : u - uq - (kind - 1) * uk) * HPW;
    return min((kind == 0 ? a.Hq : a.Hkv) - h0, HPW);
  };
  auto ask = [&](u32x4 (&raw)[AHEAD], int first) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      int kind, h0;
      const int u = first + k * step, heads = unit(u, kind, h0);
      raw[k] = u32x4{0u, 0u, 0u, 0u};
      if (u < units && token && sub < heads && in_head)
        raw[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + ((kind == 0 ? 0 : a.Hq + (kind - 1) * a.Hkv) + h0) * dh + in_unit));
    }
  };
  const int first0 = TB > 1 ? wave % TW : wave + 4 * blockIdx.y;
  ask(raw, first0);  // (on their way while the angles are formed)
  for (int i = threadIdx.x; i < TB * pairs; i += THREADS) {
    const int t = TB > 1 ? i / pairs : 0, j = i - t * pairs;
    if (n0 + t < a.N) {
      double sn = 0.0, cs = 1.0;
      if (j < half) turn_of(a.positions[n0 + t], a.inv_freq[j], sn, cs);
      turns[i] = double2{cs, sn};
      turns32[i] = float2{(float)cs, (float)sn};
    }
  }
  if (threadIdx.x < TB) {
    const int m = n0 + threadIdx.x;
    const long long s = m < a.N && a.codes != nullptr ? a.slots[m] : -1;
    const int slot = s >= 0 && s < a.num_slots ? (int)s : -1;
    const int page = slot < 0 ? 0 : slot / a.ps, off = slot < 0 ? 0 : slot - page * a.ps;
    slot_of[threadIdx.x] = slot;
    const size_t rows = (size_t)page * a.Hkv * 2 * a.ps;
    code_at[threadIdx.x] = (rows + (off & ~15)) * dh;
    scales_at[threadIdx.x] = rows + off;
    temper[threadIdx.x] = a.floor_scale > 0.f && m < a.N
                              ? 1.0f + a.attn_scale * log1pf(floorf(((float)a.positions[m] + 1.0f) / a.floor_scale)) : 1.f;
  }
  __syncthreads();

  const int slot = slot_of[tk];
  const size_t plane_codes = (size_t)a.ps * dh, at = code_at[tk], scale_at = scales_at[tk];
  for (int first = first0; token && first < units; first += AHEAD * step) {
    ask(next, first + AHEAD * step);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int u = first + k * step;
      if (u >= units) break;
      int kind, h0;
      const bool live = sub < unit(u, kind, h0) && in_head;
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(raw[k][i] << 16);
        x[2 * i + 1] = __uint_as_float(raw[k][i] & 0xffff0000u);
      }
      if (kind == 0) {
        prepare_head<float, LPH>(x, a, a.norm_wq, l, live, turns32 + tk * pairs);
        const float mul = temper[tk];
        if (live) {
          const u32x4 v = u32x4{pack_bf16(x[0] * mul, x[1] * mul), pack_bf16(x[2] * mul, x[3] * mul), pack_bf16(x[4] * mul, x[5] * mul),
                    pack_bf16(x[6] * mul, x[7] * mul)};
          u32x4* dst = reinterpret_cast<u32x4*>(a.q_out + ((size_t)n * a.Hq + h0) * dh + in_unit);
          if (TW == 1 && TB > 1) __builtin_nontemporal_store(v, dst);
          else *dst = v;
        }
        continue;
      }
      if (kind == 1) {
        double y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i];
        prepare_head<double, LPH>(y, a, a.norm_wk, l, live, turns + tk * pairs);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = toward_odd(y[i]);
      }
      uint32_t top = 0;  // the row's largest magnitude, as bits (what is no number is beyond all)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
      for (int o = LPH >> 1; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      if (!live || slot < 0) continue;
      const int byte = scale_byte(top), plane = 2 * (h0 + sub) + kind - 1;
      const float f = code_factor(byte);
      u32x2 c = {kCodesNaN, kCodesNaN};
      if (byte < 255) c = u32x2{pack_codes(x[0] * f, x[1] * f, x[2] * f, x[3] * f), pack_codes(x[4] * f, x[5] * f, x[6] * f, x[7] * f)};
      if (l == 0) a.scales[scale_at + (size_t)plane * a.ps] = (uint8_t)(byte < 255 ? byte : 127);
      if (TB > 1) {
        *reinterpret_cast<u32x2*>(held + ((kind - 1) * TB + tk) * row_codes + h0 * dh + in_unit) = c;
      } else {
        uint8_t* block = a.codes + at + plane * plane_codes;
        if (kind == 1) {
          *reinterpret_cast<u32x2*>(block + key_place(8 * l, slot & 15, dh)) = c;
        } else {
          uint8_t* dst = block + value_place(8 * l, slot & 15, dh);
          const int u2 = lane_codes(8 * l, dh);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i * u2] = (uint8_t)((i < 4 ? c[0] : c[1]) >> (8 * (i & 3)));
        }
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) raw[k] = next[k];
  }
  if (TB == 1 || a.codes == nullptr) return;

  // rows that begin an aligned four of a page that the block fills (2), that belong to one (1), others (0)
  if (threadIdx.x < TB) {
    const int r = threadIdx.x;
    int lead = 0;
#pragma unroll
    for (int back = 0; back < 4; ++back) {
      const int b = r - back;
      if (b < 0 || b + 3 >= TB) continue;
      const int s = slot_of[b];
      if (s >= 0 && (s & 3) == 0 && slot_of[b + 1] == s + 1 && slot_of[b + 2] == s + 2 && slot_of[b + 3] == s + 3)
        lead = max(lead, back == 0 ? 2 : 1);
    }
    leads[r] = lead;
  }
  __syncthreads();
  {  // keys: eight codes, tokens next to each other
    const int t = threadIdx.x % TB, mine = slot_of[t], chunks = dh / 8;
    uint8_t* page = a.codes + code_at[t];
    if (mine >= 0)
      for (int i = threadIdx.x / TB; i < a.Hkv * chunks; i += THREADS / TB) {
        const int h = over(i, a.key_chunks), c = i - h * chunks;
        *reinterpret_cast<u32x2*>(page + 2 * h * plane_codes + key_place(8 * c, mine & 15, dh)) =
            *reinterpret_cast<const u32x2*>(held + t * row_codes + h * dh + 8 * c);
      }
  }
  const int quads = (int)a.value_quads.d;  // (piece, element % 16) pairs of a head
  for (int i = threadIdx.x; i < a.Hkv * quads; i += THREADS) {
    const int h = over(i, a.value_quads), e = i - h * quads;
    const int d = e / 16 * 64 + (e & 15), u = lane_codes(d, dh);
#pragma unroll 2
    for (int t = 0; t < TB; ++t) {
      const int mine = slot_of[t], lead = leads[t];
      if (mine < 0 || lead == 1) continue;
      const uint8_t* row = held + (TB + t) * row_codes + h * dh + d;
      uint8_t* dst = a.codes + code_at[t] + (2 * h + 1) * plane_codes + value_place(d, mine & 15, dh);
      if (lead == 2) {
        u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * j < u)
            v[j] = row[16 * j] | row[row_codes + 16 * j] << 8 | row[2 * row_codes + 16 * j] << 16 |
                   (uint32_t)row[3 * row_codes + 16 * j] << 24;
        if (u == 16) *reinterpret_cast<u32x4*>(dst) = v;
        else *reinterpret_cast<u32x2*>(dst) = u32x2{v[0], v[1]};
      } else {
        for (int j = 0; 4 * j < u; ++j) dst[4 * j] = row[16 * j];
      }
    }
  }
}

// Pages in bfloat16, in the layout of the attention kernels (keys [page_size][dh], values [dh][page_size]; exact wherever
// bfloat16 holds the number: not below 2^-126, nor a code times its scale of 2^128).  Page i is page_ids[where[i]] (where null: page_ids[i]); an id that is no page's gives NaN.  An item is 16 bytes of
// the result: eight elements of a key, or eight keys of an element of the values; blockIdx: (page, part of its items, keys or
// values), and a page's items follow each other in the result's order, so that every store of a wavefront is one kilobyte.
// codes, scales, page_heads: of the first of the Hkv heads that are read, in pages of page_heads.
// attend: for attention, whose tiles share the values of keys that some of their queries do not see (zero times NaN is NaN): a
// row of values that is NaN is read as zero, and its key as NaN, which a mask takes away from the queries that do not see it.
// Memory bounds it: 32,768 tokens of 8 x 128 31 us, 6.5 TB/s, with stores that the caches need not keep (with others 37 to 46).
constexpr int kReadItems = 4;  // of a thread
__device__ __forceinline__ uint32_t two_bf16(uint32_t w, float scale, bool hi) {
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
__global__ __launch_bounds__(256) void quantized_read_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             const int* __restrict__ page_ids,
                                                             const int* __restrict__ where, bf16_t* __restrict__ out,
                                                             int num_pages, int attend, int page_heads, int Hkv, int ps, int dh, Divisor plane_items,
                                                             Divisor row_keys, Divisor row_values) {
  const int i = blockIdx.x, which = blockIdx.z;
  const int page = page_ids[where != nullptr ? where[i] : i];
  const bool ok = page >= 0 && page < num_pages;
  const int items = Hkv * (int)plane_items.d;
  const size_t plane_codes = (size_t)ps * dh;
  const uint8_t* cp = codes + ((size_t)(ok ? page : 0) * page_heads * 2 + which) * plane_codes;  // head h: + 2 h planes
  const uint8_t* sp = scales + ((size_t)(ok ? page : 0) * page_heads * 2 + which) * ps;
  bf16_t* dst = out + ((size_t)i * 2 + which) * Hkv * plane_codes;
  const int first = blockIdx.y * (256 * kReadItems) + threadIdx.x;
  u32x2 c[kReadItems], f[kReadItems];
  uint32_t value[kReadItems] = {};  // attend: a code of the key's values
#pragma unroll
  for (int k = 0; k < kReadItems; ++k) {  // everything is asked for before the first item is worked on
    const int at = min(first + 256 * k, items - 1);
    const int h = over(at, plane_items), r = at - h * (int)plane_items.d;
    const uint8_t* plane = cp + 2 * h * plane_codes;
    const uint8_t* row_scales = sp + 2 * h * ps;
    if (which == 0) {
      const int key = over(r, row_keys), d = 8 * (r - key * (int)row_keys.d);
      c[k] = *reinterpret_cast<const u32x2*>(plane + (key & ~15) * dh + key_place(d, key & 15, dh));
      f[k][0] = row_scales[key];
      if (attend) value[k] = plane[plane_codes + (key & ~15) * dh + value_place(0, key & 15, dh)];
    } else {
      const int d = over(r, row_values), key = 8 * (r - d * (int)row_values.d);
      const uint8_t* p = plane + (key & ~15) * dh + value_place(d, key & 15, dh);
      c[k][0] = *reinterpret_cast<const uint32_t*>(p);
      c[k][1] = *reinterpret_cast<const uint32_t*>(p + 16 * lane_codes(d, dh));
      f[k] = *reinterpret_cast<const u32x2*>(row_scales + key);
    }
  }
#pragma unroll
  for (int k = 0; k < kReadItems; ++k) {
    const int at = first + 256 * k;
    if (at >= items) break;
    u32x4 v;
    if (which == 0) {
      const float s = scale_of(f[k][0]);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = two_bf16(c[k][j >> 1], s, j & 1);
      if ((value[k] & 0x7fu) == 0x7fu) v = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    } else {
      if (attend) {
#pragma unroll
        for (int j = 0; j < 2; ++j) c[k][j] &= ~codes_none(c[k][j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto x = (j & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)c[k][j >> 1], true)
                               : __builtin_amdgcn_cvt_pk_f32_fp8((int)c[k][j >> 1], false);
        const uint32_t b = f[k][j >> 1] >> (16 * (j & 1));
        v[j] = pack_bf16(x[0] * scale_of(b & 255u), x[1] * scale_of((b >> 8) & 255u));
      }
    }
    if (!ok) v = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(dst + 8 * (size_t)at));
  }
}

static bool sizes_ok(int dh, int Hq, int Hkv, int ps) {
  return quantized_head_ok(dh) && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 32 && ps >= 16 && ps % 16 == 0;
}

JLE_API int jle_quantized_prepare(const void* qkv, void* q_out, void* codes, void* scales, const int* positions,
                                  const int* slot_mapping, const float* inv_freq, float norm_eps, int norm_first,
                                  const float* norm_wq, const float* norm_wk, int pairing, int rotary_dim,
                                  float floor_scale, float attn_scale, int N, int Hq, int Hkv, int dh, int ps,
                                  int num_pages, int* clear, int num_clear, hipStream_t s) {
  if (N <= 0) return 0;
  if (!sizes_ok(dh, Hq, Hkv, ps) || num_pages < 0) return JLE_BAD_ARG;
  if ((codes == nullptr) != (scales == nullptr) || (codes != nullptr && slot_mapping == nullptr)) return JLE_BAD_ARG;
  if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)codes) & 15) return JLE_BAD_ARG;
  if (num_clear < 0 || (num_clear > 0 && clear == nullptr) || (long long)num_pages * ps > 0x7fffffffll) return JLE_BAD_ARG;
  if (inv_freq == nullptr) rotary_dim = 0;
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > dh || (pairing != 0 && pairing != 1)) return JLE_BAD_ARG;
  if (pairing == 1 && rotary_dim % 16) return JLE_BAD_ARG;
  const int lph = dh == 32 ? 4 : dh == 64 ? 8 : dh == 256 ? 32 : 16;
  const int pairs = inv_freq == nullptr ? 0 : pairing == 0 ? dh / 2 : rotary_dim / 2;
  const PrepareArgs a = {(const bf16_t*)qkv, (bf16_t*)q_out, (uint8_t*)codes, (uint8_t*)scales, positions, slot_mapping,
                         inv_freq, norm_wq, norm_wk, norm_eps, 1.0 / dh, floor_scale, attn_scale, norm_first, pairs, pairing, rotary_dim,
                         N, Hq, Hkv, dh, ps, (long long)num_pages * ps, divisor(dh / 8), divisor((dh + 63) / 64 * 16),
                         clear, num_clear};
  const int hpw = 64 / lph;
  const int units = (Hq + hpw - 1) / hpw + (codes != nullptr ? 2 * ((Hkv + hpw - 1) / hpw) : 0);
  // Several tokens a block from kManyTokens on, where their codes fit a quarter of the shared memory: with the whole head turned
  // up to 14 kv heads of 128, 32 of 64, 4 of 256.  With more, one token a block at any number, whose values are stored code by
  // code (2,048 tokens of 32 heads of 128 with 8, 16 and 32 kv heads: 24, 44 and 63 us; 8,191 with 8 and 32: 55 and 207).
  const size_t turns = (size_t)pairs * (sizeof(double2) + sizeof(float2));
  const size_t lds = kTokens * (turns + 2 * (size_t)Hkv * dh);
  const bool many = N >= kManyTokens && lds <= 40 * 1024;
  // two wavefronts a token while the blocks of eight are no more than two a compute unit (2,048 tokens of 40 + 16 heads 17.8 ->
  // 15.6 us, 8,191 of 32 + 16 49 -> 60)
  const bool wide = N <= 2 * 256 * kTokens;
#define LAUNCH(LPH)                                                                                                        \
  do {                                                                                                                     \
    const dim3 blocks((N + kTokens - 1) / kTokens);                                                                        \
    if (many && wide)                                                                                                      \
      hipLaunchKernelGGL((quantized_prepare_kernel<LPH, kTokens, 2>), blocks, dim3(kTokens * 128), lds, s, a);             \
    else if (many)                                                                                                         \
      hipLaunchKernelGGL((quantized_prepare_kernel<LPH, kTokens, 1>), blocks, dim3(kTokens * 64), lds, s, a);              \
    else                                                                                                                   \
      hipLaunchKernelGGL((quantized_prepare_kernel<LPH, 1, 1>), dim3(N, (units + 3) / 4), dim3(256), turns, s, a);         \
  } while (0)
  switch (lph) {
    case 4: LAUNCH(4); break;
    case 8: LAUNCH(8); break;
    case 16: LAUNCH(16); break;
    case 32: LAUNCH(32); break;
  }
#undef LAUNCH
  JLE_LAUNCH_CHECK();
  return 0;
}

JLE_API int jle_quantized_read(const void* codes, const void* scales, const int* page_ids, const int* where, void* out,
                               int n, int num_pages, int attend, int page_heads, int first_head, int Hkv, int dh, int ps,
                               hipStream_t s) {
  if (n <= 0) return 0;
  if (!sizes_ok(dh, Hkv, Hkv, ps) || num_pages <= 0) return JLE_BAD_ARG;
  if (first_head < 0 || first_head > page_heads - Hkv) return JLE_BAD_ARG;
  if (((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)out) & 15) return JLE_BAD_ARG;
  const long long items = (long long)Hkv * ps * (dh / 8);
  const long long parts = (items + 256 * kReadItems - 1) / (256 * kReadItems);
  if (parts > 65535) return JLE_BAD_ARG;
  hipLaunchKernelGGL(quantized_read_kernel, dim3(n, (unsigned)parts, 2), dim3(256), 0, s,
                     (const uint8_t*)codes + (size_t)first_head * 2 * ps * dh, (const uint8_t*)scales + (size_t)first_head * 2 * ps,
                     page_ids, where, (bf16_t*)out, num_pages, attend, page_heads, Hkv, ps, dh, divisor(ps * (dh / 8)),
                     divisor(dh / 8), divisor(ps / 8));
  JLE_LAUNCH_CHECK();
  return 0;
}
