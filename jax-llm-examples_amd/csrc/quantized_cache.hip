// A cache in 8 bits is written and read back (the format: quantized.h).
//
// Writing follows the fused q|k|v projection: rms norm of q and k over the head (with or without weights, before or after
// the rotation), rotary embedding (adjacent or half-split pairs, over the head's leading part), position-dependent query
// scale, as attention_prep.hip has them, and k and v rounded once, from float32, to codes and a scale byte a row.
#include "quantized.h"

using namespace jle;

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

// LPH lanes a head (a power of two, at least dh / 8), eight neighbouring elements a lane, 64 / LPH heads a wavefront.
template <int LPH>
__global__ __launch_bounds__(256) void quantized_prepare_kernel(
    const bf16_t* __restrict__ qkv, bf16_t* __restrict__ q_out, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
    const int* __restrict__ positions, const int* __restrict__ slot_mapping, const float* __restrict__ inv_freq,
    float norm_eps, int norm_first, const float* __restrict__ norm_wq, const float* __restrict__ norm_wk, int pairing,
    int rotary_dim, float floor_scale, float attn_scale, int N, int Hq, int Hkv, int dh, int ps, long long num_slots) {
  constexpr int HPW = 64 / LPH;
  const int lane = threadIdx.x & 63;
  const int H = Hq + 2 * Hkv;
  const int per_token = (H + HPW - 1) / HPW;
  const long long item = (long long)blockIdx.x * 4 + wave_index();
  const int n = (int)(item / per_token);
  if (n >= N) return;
  const int l = lane & (LPH - 1);
  const int h = (int)(item - (long long)n * per_token) * HPW + lane / LPH;
  const bool live = h < H && 8 * l < dh;
  const bool is_q = h < Hq, is_v = h >= Hq + Hkv;
  const int pos = positions[n];
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (live) {
    const u32x4 r = *reinterpret_cast<const u32x4*>(qkv + ((size_t)n * H + h) * dh + 8 * l);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(r[i] << 16);
      x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
  const float* w = is_q ? norm_wq : norm_wk;
  float wt[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) wt[i] = (live && !is_v && w != nullptr) ? w[8 * l + i] : 1.f;
  auto over_head = [&](float s) {
#pragma unroll
    for (int o = LPH >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    return s;
  };
  auto norm = [&]() {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
    ss = over_head(ss);
    if (is_v) return;
    const float mul = 1.0f / sqrtf(ss / (float)dh + norm_eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= mul * wt[i];
  };
  if (norm_eps >= 0.f && norm_first) norm();
  if (inv_freq != nullptr) {
    if (pairing == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * l + i;
        if (2 * j < rotary_dim && !is_v) {
          const float ang = (float)pos * inv_freq[j];
          const float sn = sinf(ang), cs = cosf(ang);
          const float a = x[2 * i], b = x[2 * i + 1];
          x[2 * i] = a * cs - b * sn;
          x[2 * i + 1] = b * cs + a * sn;
        }
      }
    } else {  // (half of the rotated part is a multiple of 8: a lane's partners are all in one other lane)
      const int half = rotary_dim >> 1;
      const bool turned = 8 * l < rotary_dim, leading = 8 * l < half;
      const int other = turned ? (leading ? lane + half / 8 : lane - half / 8) : lane;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], other, 64);
      if (turned && !is_v && live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float ang = (float)pos * inv_freq[leading ? 8 * l + i : 8 * l + i - half];
          const float sn = sinf(ang), cs = cosf(ang);
          x[i] = leading ? x[i] * cs - y[i] * sn : x[i] * cs + y[i] * sn;
        }
      }
    }
  }
  if (norm_eps >= 0.f && !norm_first) norm();
  uint32_t top = 0;  // the row's largest magnitude, as bits (what is no number is beyond all)
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = LPH >> 1; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if (!live) return;
  if (is_q) {
    if (floor_scale > 0.f) {
      const float mul = 1.0f + attn_scale * log1pf(floorf(((float)pos + 1.0f) / floor_scale));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= mul;
    }
    *reinterpret_cast<u32x4*>(q_out + ((size_t)n * Hq + h) * dh + 8 * l) =
        u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
    return;
  }
  if (codes == nullptr) return;
  const long long slot = slot_mapping[n];
  if (slot < 0 || slot >= num_slots) return;
  const int byte = scale_byte(top);
  const float f = code_factor(byte);
  uint32_t c0 = kCodesNaN, c1 = kCodesNaN;
  if (byte < 255) {
    c0 = pack_codes(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
    c1 = pack_codes(x[4] * f, x[5] * f, x[6] * f, x[7] * f);
  }
  const long long page = slot / ps;
  const int off = (int)(slot - page * ps);
  const size_t plane = ((size_t)page * Hkv + (is_v ? h - Hq - Hkv : h - Hq)) * 2 + (is_v ? 1 : 0);
  uint8_t* block = codes + (plane * ps + (off & ~15)) * dh;
  if (l == 0) scales[plane * ps + off] = (uint8_t)(byte < 255 ? byte : 127);
  if (is_v) {
    uint8_t* dst = block + value_place(8 * l, off & 15, dh);
    const int u = lane_codes(8 * l, dh);
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i * u] = (uint8_t)((i < 4 ? c0 >> (8 * i) : c1 >> (8 * (i - 4))));
  } else {
    *reinterpret_cast<u32x2*>(block + key_place(8 * l, off & 15, dh)) = u32x2{c0, c1};
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
                                  int num_pages, hipStream_t s) {
  if (N <= 0) return 0;
  if (!jle_quantized_supported(dh, Hq, Hkv, ps) || num_pages < 0) return JLE_BAD_ARG;
  if ((codes == nullptr) != (scales == nullptr) || (codes != nullptr && slot_mapping == nullptr)) return JLE_BAD_ARG;
  if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)codes) & 15) return JLE_BAD_ARG;
  if (inv_freq == nullptr) rotary_dim = 0;
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > dh || (pairing != 0 && pairing != 1)) return JLE_BAD_ARG;
  if (pairing == 1 && rotary_dim % 16) return JLE_BAD_ARG;
  const int lph = dh == 32 ? 4 : dh == 64 ? 8 : dh == 256 ? 32 : 16;
  const long long waves = (long long)N * ((Hq + 2 * Hkv + 64 / lph - 1) / (64 / lph));
  if (waves > (1ll << 32)) return JLE_BAD_ARG;
  dim3 g((unsigned)((waves + 3) / 4)), b(256);
#define LAUNCH(LPH)                                                                                                      \
  hipLaunchKernelGGL(quantized_prepare_kernel<LPH>, g, b, 0, s, (const bf16_t*)qkv, (bf16_t*)q_out, (uint8_t*)codes,     \
                     (uint8_t*)scales, positions, slot_mapping, inv_freq, norm_eps, norm_first, norm_wq, norm_wk,        \
                     pairing, rotary_dim, floor_scale, attn_scale, N, Hq, Hkv, dh, ps, (long long)num_pages * ps)
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
