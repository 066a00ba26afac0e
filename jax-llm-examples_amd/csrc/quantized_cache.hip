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
// in some hundred thousand falls the other way.  Queries, which are rounded to bfloat16, are worked on in float32, with the
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

struct PrepareArgs {
  const bf16_t* qkv;
  bf16_t* q_out;
  uint8_t *codes, *scales;  // null: keys and values are not written
  const int *positions, *slots;
  const float* inv_freq;  // null: no rotation
  const float *norm_wq, *norm_wk;
  float norm_eps;  // < 0: no norm
  float floor_scale, attn_scale;
  int norm_first, pairing, rotary_dim;  // pairing 0: (x[2j], x[2j + 1]), 1: (x[j], x[j + rotary_dim / 2])
  int N, Hq, Hkv, dh, ps;
  long long num_slots;
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

// A head's numbers, eight a lane (l: the lane's place in the head), normed and turned.  F: what is computed in.
template <typename F, int LPH>
__device__ __forceinline__ void prepare_head(F (&x)[8], const PrepareArgs& a, const float* w, int l, bool live, const double2* turns) {
  auto norm = [&]() {
    F ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma(x[i], x[i], ss);
    ss = over_head<F, LPH>(ss);
    const F mul = F(1) / sqrt(ss / (F)a.dh + (F)a.norm_eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= w != nullptr && live ? mul * (F)w[8 * l + i] : mul;
  };
  if (a.norm_eps >= 0.f && a.norm_first) norm();
  if (a.inv_freq != nullptr) {
    if (a.pairing == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (8 * l + 2 * i < a.rotary_dim) {
          const double2 t = turns[4 * l + i];  // (cosine, sine)
          const F p = x[2 * i], q = x[2 * i + 1], c = (F)t.x, s = (F)t.y;
          x[2 * i] = fma(p, c, -(q * s));
          x[2 * i + 1] = fma(q, c, p * s);
        }
      }
    } else {  // (half of the rotated part is a multiple of 8: a lane's partners are all in one other lane)
      const int half = a.rotary_dim >> 1, lane = threadIdx.x & 63;
      const bool turned = 8 * l < a.rotary_dim, leading = 8 * l < half;
      const int other = turned ? (leading ? lane + half / 8 : lane - half / 8) : lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const F y = __shfl(x[i], other, 64);
        if (turned) {
          const double2 t = turns[leading ? 8 * l + i : 8 * l + i - half];
          x[i] = fma(x[i], (F)t.x, (leading ? -y : y) * (F)t.y);
        }
      }
    }
  }
  if (a.norm_eps >= 0.f && !a.norm_first) norm();
}

// A block takes TB consecutive tokens; LPH lanes a head (a power of two, at least dh / 8), eight neighbouring elements a lane,
// 64 / LPH heads of a kind (queries, keys, values) a wavefront at a time: a *unit*.  The block's sines and cosines are formed
// once.  With one token a block (few tokens) the units are shared out among gridDim.y blocks and the codes go straight into
// their pages; with several the codes are gathered in shared memory and written in pieces of 16 bytes: keys a token's sixteen
// elements, values the four keys of four elements where the block's tokens fill an aligned four of a page (other values byte
// by byte).
template <int LPH, int TB>
__global__ __launch_bounds__(256) void quantized_prepare_kernel(PrepareArgs a) {
  constexpr int HPW = 64 / LPH;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int l = lane & (LPH - 1), sub = lane / LPH;
  const int n0 = blockIdx.x * TB, half = a.rotary_dim >> 1;
  const int H = a.Hq + 2 * a.Hkv, dh = a.dh, row_codes = a.Hkv * dh;
  double2* turns = reinterpret_cast<double2*>(smem);         // [TB][half]
  uint8_t* held = smem + (size_t)TB * half * sizeof(double2);  // [2][TB][Hkv][dh], several tokens only
  __shared__ int slot_of[TB], leads[TB];
  if (a.num_clear > 0 && blockIdx.y == 0)
    for (int i = blockIdx.x * 256 + threadIdx.x; i < a.num_clear; i += gridDim.x * 256) a.clear[i] = 0;

  const int uq = (a.Hq + HPW - 1) / HPW, uk = a.codes != nullptr ? (a.Hkv + HPW - 1) / HPW : 0;
  const int units = uq + 2 * uk, all = TB * units;
  const int stride = 4 * gridDim.y;
  const bool in_head = 8 * l < dh;
  constexpr int AHEAD = TB > 1 ? 4 : 1;  // units' rows asked for at once
  for (int i = threadIdx.x; i < TB * half; i += 256) {
    const int tk = i / half;
    if (n0 + tk < a.N) {
      double sn, cs;
      turn_of(a.positions[n0 + tk], a.inv_freq[i - tk * half], sn, cs);
      turns[i] = double2{cs, sn};
    }
  }
  if (TB > 1 && threadIdx.x < TB) {
    const int n = n0 + threadIdx.x;
    long long s = n < a.N && a.codes != nullptr ? a.slots[n] : -1;
    slot_of[threadIdx.x] = s >= 0 && s < a.num_slots ? (int)s : -1;
  }
  __syncthreads();

  for (int first = wave + 4 * blockIdx.y; first < all; first += AHEAD * stride) {
    u32x4 raw[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int at = first + k * stride, tk = at / units, u = at - tk * units;
      const int kind = u < uq ? 0 : u < uq + uk ? 1 : 2;
      const int h = (kind == 0 ? u : u - uq - (kind - 1) * uk) * HPW + sub;
      const bool live = at < all && n0 + tk < a.N && h < (kind == 0 ? a.Hq : a.Hkv) && in_head;
      raw[k] = u32x4{0u, 0u, 0u, 0u};
      if (live)
        raw[k] = *reinterpret_cast<const u32x4*>(a.qkv + ((size_t)(n0 + tk) * H + (kind == 0 ? 0 : a.Hq + (kind - 1) * a.Hkv) + h) * dh + 8 * l);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int at = first + k * stride, tk = at / units, u = at - tk * units;
      const int n = n0 + tk;
      if (at >= all || n >= a.N) continue;  // (the same in all lanes)
      const int kind = u < uq ? 0 : u < uq + uk ? 1 : 2;
      const int h = (kind == 0 ? u : u - uq - (kind - 1) * uk) * HPW + sub;
      const bool live = h < (kind == 0 ? a.Hq : a.Hkv) && in_head;
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(raw[k][i] << 16);
        x[2 * i + 1] = __uint_as_float(raw[k][i] & 0xffff0000u);
      }
      if (kind == 0) {
        prepare_head<float, LPH>(x, a, a.norm_wq, l, live, turns + tk * half);
        if (a.floor_scale > 0.f) {
          const float mul = 1.0f + a.attn_scale * log1pf(floorf(((float)a.positions[n] + 1.0f) / a.floor_scale));
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= mul;
        }
        if (live)
          *reinterpret_cast<u32x4*>(a.q_out + ((size_t)n * a.Hq + h) * dh + 8 * l) =
              u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
        continue;
      }
      if (kind == 1) {
        double y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i];
        prepare_head<double, LPH>(y, a, a.norm_wk, l, live, turns + tk * half);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)y[i];
      }
      uint32_t top = 0;  // the row's largest magnitude, as bits (what is no number is beyond all)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
      for (int o = LPH >> 1; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      if (!live) continue;
      long long slot;
      if (TB > 1) {
        slot = slot_of[tk];
      } else {
        slot = a.slots[n];
        if (slot >= a.num_slots) slot = -1;
      }
      if (slot < 0) continue;
      const int byte = scale_byte(top);
      const float f = code_factor(byte);
      u32x2 c = {kCodesNaN, kCodesNaN};
      if (byte < 255) c = u32x2{pack_codes(x[0] * f, x[1] * f, x[2] * f, x[3] * f), pack_codes(x[4] * f, x[5] * f, x[6] * f, x[7] * f)};
      const int which = kind - 1, page = (int)(slot / a.ps), off = (int)(slot - (long long)page * a.ps);
      const size_t plane = ((size_t)page * a.Hkv + h) * 2 + which;
      if (l == 0) a.scales[plane * a.ps + off] = (uint8_t)(byte < 255 ? byte : 127);
      if (TB > 1) {
        *reinterpret_cast<u32x2*>(held + (size_t)(which * TB + tk) * row_codes + h * dh + 8 * l) = c;
      } else {
        uint8_t* block = a.codes + (plane * a.ps + (off & ~15)) * dh;
        if (which == 0) {
          *reinterpret_cast<u32x2*>(block + key_place(8 * l, off & 15, dh)) = c;
        } else {
          uint8_t* dst = block + value_place(8 * l, off & 15, dh);
          const int u2 = lane_codes(8 * l, dh);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i * u2] = (uint8_t)((i < 4 ? c[0] : c[1]) >> (8 * (i & 3)));
        }
      }
    }
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
  auto block_of = [&](int slot, int h, int which) {
    const int page = slot / a.ps, off = slot - page * a.ps;
    return a.codes + ((((size_t)page * a.Hkv + h) * 2 + which) * a.ps + (off & ~15)) * dh;
  };
  const int chunks = dh / 8;
  for (int i = threadIdx.x; i < TB * a.Hkv * chunks; i += 256) {  // keys: eight codes, tokens next to each other
    const int tk = i % TB, c = i / TB % chunks, h = i / (TB * chunks);
    const int slot = slot_of[tk];
    if (slot >= 0)
      *reinterpret_cast<u32x2*>(block_of(slot, h, 0) + key_place(8 * c, slot & 15, dh)) =
          *reinterpret_cast<const u32x2*>(held + (size_t)tk * row_codes + h * dh + 8 * c);
  }
  const int quads = (dh + 63) / 64 * 16;  // (piece, element % 16) pairs
  for (int i = threadIdx.x; i < TB * a.Hkv * quads; i += 256) {
    const int e = i % quads, h = i / quads % a.Hkv, tk = i / (quads * a.Hkv);
    const int slot = slot_of[tk], lead = leads[tk];
    if (slot < 0 || lead == 1) continue;
    const int d = e / 16 * 64 + (e & 15), u = lane_codes(d, dh);
    const uint8_t* row = held + (size_t)(TB + tk) * row_codes + h * dh + d;
    uint8_t* dst = block_of(slot, h, 1) + value_place(d, slot & 15, dh);
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

// Pages in bfloat16, in the layout of the attention kernels (keys [page_size][dh], values [dh][page_size]; every number is
// exact).  A wavefront takes sixteen keys of one (page, kv head), keys or values.  Page i is page_ids[where[i]] (where null:
// page_ids[i]); an id that is no page's gives NaN.
__global__ __launch_bounds__(256) void quantized_read_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             const int* __restrict__ page_ids,
                                                             const int* __restrict__ where, bf16_t* __restrict__ out,
                                                             long long items, int num_pages, int Hkv, int ps, int dh) {
  const long long item = (long long)blockIdx.x * 4 + wave_index();
  if (item >= items) return;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int blocks = ps / 16;
  const int kb = (int)(item % blocks);
  const long long i2 = item / blocks;
  const int hk = (int)(i2 % Hkv);
  const long long i3 = i2 / Hkv;
  const int which = (int)(i3 & 1);
  const long long i = i3 >> 1;
  const int page = page_ids[where != nullptr ? where[i] : (int)i];
  const bool ok = page >= 0 && page < num_pages;
  const size_t plane = ((size_t)(ok ? page : 0) * Hkv + hk) * 2 + which;
  const uint8_t* src = codes + (plane * ps + 16 * kb) * dh;
  const uint8_t* sc = scales + plane * ps + 16 * kb;
  bf16_t* dst = out + (((size_t)i * 2 + which) * Hkv + hk) * ps * dh;
  float f[4];  // keys: the lane's one; values: its four
  if (which == 0) {
    f[0] = f[1] = f[2] = f[3] = ok ? scale_of(sc[r]) : 1.f;
  } else {
    const uint32_t b = *reinterpret_cast<const uint32_t*>(sc + 4 * g);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = ok ? scale_of((b >> (8 * j)) & 255u) : 1.f;
  }
  for (int d0 = 0; d0 < dh; d0 += 64) {
    const int u = lane_codes(d0, dh);
    uint32_t w[4] = {kCodesNaN, kCodesNaN, kCodesNaN, kCodesNaN};
    if (ok) {
      const uint8_t* p = src + d0 * 16 + lane * u;
      if (u == 16) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = v[j];
      } else {
        const u32x2 v = *reinterpret_cast<const u32x2*>(p);
        w[0] = v[0];
        w[1] = v[1];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (4 * j >= u) break;
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], true);
      const u32x2 b = {pack_bf16(lo[0] * f[0], lo[1] * f[1]), pack_bf16(hi[0] * f[2], hi[1] * f[3])};
      if (which == 0)
        *reinterpret_cast<u32x2*>(dst + (size_t)(16 * kb + r) * dh + d0 + u * g + 4 * j) = b;
      else
        *reinterpret_cast<u32x2*>(dst + (size_t)(d0 + 16 * j + r) * ps + 16 * kb + 4 * g) = b;
    }
  }
}

JLE_API int jle_quantized_supported(int dh, int Hq, int Hkv, int ps) {
  return quantized_head_ok(dh) && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 32 && ps >= 16 && ps % 16 == 0;
}

JLE_API int jle_quantized_prepare(const void* qkv, void* q_out, void* codes, void* scales, const int* positions,
                                  const int* slot_mapping, const float* inv_freq, float norm_eps, int norm_first,
                                  const float* norm_wq, const float* norm_wk, int pairing, int rotary_dim,
                                  float floor_scale, float attn_scale, int N, int Hq, int Hkv, int dh, int ps,
                                  int num_pages, int* clear, int num_clear, hipStream_t s) {
  if (N <= 0) return 0;
  if (!jle_quantized_supported(dh, Hq, Hkv, ps) || num_pages < 0) return JLE_BAD_ARG;
  if ((codes == nullptr) != (scales == nullptr) || (codes != nullptr && slot_mapping == nullptr)) return JLE_BAD_ARG;
  if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)codes) & 15) return JLE_BAD_ARG;
  if (num_clear < 0 || (num_clear > 0 && clear == nullptr) || (long long)num_pages * ps > 0x7fffffffll) return JLE_BAD_ARG;
  if (inv_freq == nullptr) rotary_dim = 0;
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > dh || (pairing != 0 && pairing != 1)) return JLE_BAD_ARG;
  if (pairing == 1 && rotary_dim % 16) return JLE_BAD_ARG;
  const int lph = dh == 32 ? 4 : dh == 64 ? 8 : dh == 256 ? 32 : 16;
  const PrepareArgs a = {(const bf16_t*)qkv, (bf16_t*)q_out, (uint8_t*)codes, (uint8_t*)scales, positions, slot_mapping,
                         inv_freq, norm_wq, norm_wk, norm_eps, floor_scale, attn_scale, norm_first, pairing, rotary_dim,
                         N, Hq, Hkv, dh, ps, (long long)num_pages * ps, clear, num_clear};
  const int hpw = 64 / lph;
  const int units = (Hq + hpw - 1) / hpw + (codes != nullptr ? 2 * ((Hkv + hpw - 1) / hpw) : 0);
  // Several tokens a block from kManyTokens on, where their codes fit a quarter of the shared memory.
  const size_t turns = (size_t)rotary_dim / 2 * sizeof(double2);
  const size_t lds = kTokens * (turns + 2 * (size_t)Hkv * dh);
  const bool many = N >= kManyTokens && lds <= 40 * 1024;
#define LAUNCH(LPH)                                                                                                     \
  do {                                                                                                                  \
    if (many)                                                                                                           \
      hipLaunchKernelGGL((quantized_prepare_kernel<LPH, kTokens>), dim3((N + kTokens - 1) / kTokens), dim3(256), lds, s, a); \
    else                                                                                                                \
      hipLaunchKernelGGL((quantized_prepare_kernel<LPH, 1>), dim3(N, (units + 3) / 4), dim3(256), turns, s, a);          \
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
                               int n, int num_pages, int Hkv, int dh, int ps, hipStream_t s) {
  if (n <= 0) return 0;
  if (!jle_quantized_supported(dh, Hkv, Hkv, ps) || num_pages <= 0) return JLE_BAD_ARG;
  if (((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)out) & 15) return JLE_BAD_ARG;
  const long long items = (long long)n * 2 * Hkv * (ps / 16);
  if (items > (1ll << 32)) return JLE_BAD_ARG;
  hipLaunchKernelGGL(quantized_read_kernel, dim3((unsigned)((items + 3) / 4)), dim3(256), 0, s, (const uint8_t*)codes,
                     (const uint8_t*)scales, page_ids, where, (bf16_t*)out, items, num_pages, Hkv, ps, dh);
  JLE_LAUNCH_CHECK();
  return 0;
}
