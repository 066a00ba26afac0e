// Attention over a cache in 8 bits (quantized.h) for steps of single tokens and of a few tokens a request.
//
// A *tile* is a few consecutive tokens of one segment; with the query heads that share a kv head they are the tile's
// *columns*, up to 16 * CT of them.  A block takes a range of `range` key positions of one (tile, kv head); its wavefronts take
// the range's steps of 32 keys in turn, so that all of them work however short the range is.  As in attention_mfma.hip
// everything is kept transposed:
//
//   S^T[key, col] = K[key, :] . Q[col, :]        A = keys (each lane: one key, so its scale rides in the conversion to
//                                                 bfloat16, which is exact), B = queries
//   O^T[d, col]  += V^T[d, key] . P^T[key, col]   A = values (codes as they are), B = probabilities times the keys' scales
//
// The pages hold the codes in the lanes' order, so every load of a wavefront is a contiguous kilobyte.  A wavefront has two
// steps in registers or on their way.  What bounds it is memory: 2 * dh + 2 bytes a key and kv head.
//
// The wavefronts' (maximum, sum, unnormalised O^T) are merged in shared memory; with more than one range a (tile, kv head)
// the blocks' results go through memory and a second kernel merges them in order.  Which ranges there are depends on the
// position, the retention rule and `range` alone.
#include "mfma_attention.h"
#include "quantized.h"

using namespace jle;

__device__ __forceinline__ int first_key(int mode, int param, int pos) {
  if (mode == 1) return (pos / param) * param;
  if (mode == 2) return pos - param + 1 > 0 ? pos - param + 1 : 0;
  return 0;
}

template <int DH>
struct QuantizedStep {  // 32 keys of one kv head
  static constexpr int P = DH / 64;                // pieces of 64 elements
  static constexpr bool T = DH % 64 != 0;          // a last piece of 32
  u32x4 k[2][P > 0 ? P : 1], v[2][P > 0 ? P : 1];
  u32x2 kt[2], vt[2];
  uint32_t ks[2], vs[2];  // scale bytes: of the lane's key; of its four keys
  int have;               // bit tt: the tile of sixteen keys exists
};

__device__ __forceinline__ uint32_t two_codes(uint32_t w, float scale, bool hi) {
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
__device__ __forceinline__ bf16x8 eight_codes(uint32_t a, uint32_t b, float scale) {
  const u32x4 r = {two_codes(a, scale, false), two_codes(a, scale, true), two_codes(b, scale, false), two_codes(b, scale, true)};
  return __builtin_bit_cast(bf16x8, r);
}

template <int DH, int CT, int W>
__global__ __launch_bounds__(W * 64, W / 4) void attention_quantized_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
    bf16_t* __restrict__ out, float* __restrict__ ws_ml, float* __restrict__ ws_o, const int* __restrict__ positions,
    const int* __restrict__ token_segment, const int* __restrict__ block_table, int table_width, int num_pages,
    const int* __restrict__ tiles, int ranges, int range, int ret_mode, int ret_param, float scale_log2, int Hq, int Hkv,
    int ps, int max_cols) {
  using Step = QuantizedStep<DH>;
  constexpr int P = Step::P, DT = DH / 16, KC = DH / 32, LD = DH + 4;
  extern __shared__ __attribute__((aligned(16))) float smem[];  // [W][max_cols][LD], then [W][max_cols][2]
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int c16 = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % Hkv;
  const int rng = (blockIdx.x / Hkv) % ranges;
  const int tile = blockIdx.x / (Hkv * ranges);
  const int n0 = tiles[2 * tile], nt = tiles[2 * tile + 1];
  const int p_first = positions[n0], p_last = p_first + nt - 1;
  const int first = first_key(ret_mode, ret_param, p_first);
  const int r_abs = first / range + rng;
  if (r_abs > p_last / range) return;  // (this tile has fewer ranges)
  const int k_lo = max(first, r_abs * range), k_hi = min(p_last, r_abs * range + range - 1);
  const int full_lo = max(k_lo, first_key(ret_mode, ret_param, p_last)), full_hi = min(k_hi, p_first);
  const int G = Hq / Hkv, cols = nt * G;
  const int* table = block_table + (size_t)token_segment[n0] * table_width;

  int lo[CT], hi[CT];
  bf16x8 qb[CT][KC];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = ct * 16 + c16;
    const int t = c < cols ? c / G : 0, head = hk * G + (c < cols ? c - t * G : 0);
    lo[ct] = max(k_lo, first_key(ret_mode, ret_param, p_first + t));
    hi[ct] = min(k_hi, p_first + t);
    const bf16_t* row = q + ((size_t)(n0 + t) * Hq + head) * DH;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      qb[ct][2 * p] = *reinterpret_cast<const bf16x8*>(row + 64 * p + 16 * g);
      qb[ct][2 * p + 1] = *reinterpret_cast<const bf16x8*>(row + 64 * p + 16 * g + 8);
    }
    if (Step::T) qb[ct][KC - 1] = *reinterpret_cast<const bf16x8*>(row + 64 * P + 8 * g);
  }
  float m[CT], l[CT];
  f32x4 acc[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bool bad = false;

  auto load = [&](Step& s, int step) {
    s.have = 0;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int key0 = 32 * step + 16 * tt;
      int page = -1, off = 0;
      if (key0 <= k_hi && key0 + 15 >= k_lo) {
        const int idx = key0 / ps;
        off = key0 - idx * ps;
        page = idx < table_width ? table[idx] : -1;
        if (page < 0 || page >= num_pages) {
          bad = true;  // (the tile is left out, and the result is NaN)
          page = -1;
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        s.k[tt][p] = u32x4{0u, 0u, 0u, 0u};
        s.v[tt][p] = u32x4{0u, 0u, 0u, 0u};
      }
      s.kt[tt] = s.vt[tt] = u32x2{0u, 0u};
      s.ks[tt] = s.vs[tt] = 0u;
      if (page < 0) continue;
      s.have |= 1 << tt;
      const size_t plane = ((size_t)page * Hkv + hk) * 2;
      const uint8_t* kp = codes + (plane * ps + off) * DH;
      const uint8_t* vp = kp + (size_t)ps * DH;
      const uint8_t* sp = scales + plane * ps + off;
      s.ks[tt] = sp[c16];
      s.vs[tt] = *reinterpret_cast<const uint32_t*>(sp + ps + 4 * g);
#pragma unroll
      for (int p = 0; p < P; ++p) s.k[tt][p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + 1024 * p) + lane);
      if (Step::T) s.kt[tt] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(kp + 1024 * P) + lane);
#pragma unroll
      for (int p = 0; p < P; ++p) s.v[tt][p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp + 1024 * p) + lane);
      if (Step::T) s.vt[tt] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vp + 1024 * P) + lane);
    }
  };

  auto work = [&](Step& s, int step) {
    f32x4 st[CT][2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const float f = scale_of(s.ks[tt]);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) st[ct][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const bool tail = Step::T && c == KC - 1;
        const bf16x8 a = tail ? eight_codes(s.kt[tt][0], s.kt[tt][1], f)
                              : eight_codes(s.k[tt][c / 2][2 * (c & 1)], s.k[tt][c / 2][2 * (c & 1) + 1], f);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) st[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qb[ct][c], st[ct][tt], 0, 0, 0);
      }
    }
    const bool full = s.have == 3 && 32 * step >= full_lo && 32 * step + 31 <= full_hi;
    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
    if (!full) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        keep[tt] = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = 32 * step + 16 * tt + 4 * g + i;
          const bool there = (s.have >> tt & 1) != 0;
          // values and scales of keys outside the range may never have been written: they are read as zero
          if (there && key >= k_lo && key <= k_hi) keep[tt] |= 255u << (8 * i);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            if (!(there && key >= lo[ct] && key <= hi[ct])) st[ct][tt][i] = -INFINITY;
        }
        s.vs[tt] &= keep[tt];
      }
    }
    float vf[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) vf[j] = scale_of((s.vs[j >> 2] >> (8 * (j & 3))) & 255u);
    bf16x8 pb[CT];
    float corr[CT];
    bool unchanged = true;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, st[ct][j >> 2][j & 3]);
      mx = column_max(mx);
      const float m_new = fmaxf(m[ct], mx * scale_log2);  // (the scale is positive)
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      corr[ct] = __builtin_amdgcn_exp2f(m[ct] - m_use);
      unchanged = unchanged && m_new == m[ct];
      float sum = 0.f, p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(fmaf(st[ct][j >> 2][j & 3], scale_log2, -m_use));
        sum += p[j];
        p[j] *= vf[j];
      }
      l[ct] = l[ct] * corr[ct] + sum;
      m[ct] = m_new;
      const u32x4 pk = {pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7])};
      pb[ct] = __builtin_bit_cast(bf16x8, pk);
    }
    if (!__all(unchanged)) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[ct][dt][i] *= corr[ct];
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const bool tail = Step::T && dt >= 4 * P;
      const uint32_t w0 = (tail ? s.vt[0][dt & 1] : s.v[0][dt / 4][dt & 3]) & keep[0];
      const uint32_t w1 = (tail ? s.vt[1][dt & 1] : s.v[1][dt / 4][dt & 3]) & keep[1];
      const bf16x8 a = eight_codes(w0, w1, 1.0f);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[ct], acc[ct][dt], 0, 0, 0);
    }
  };

  const int last = k_hi / 32;
  int step = k_lo / 32 + wave;
  Step a, b;
  if (step <= last) load(a, step);
  if (step + W <= last) load(b, step + W);
  while (step <= last) {
    work(a, step);
    if (step + 2 * W <= last) load(a, step + 2 * W);
    step += W;
    if (step > last) break;
    work(b, step);
    if (step + 2 * W <= last) load(b, step + 2 * W);
    step += W;
  }
  bad = __any(bad);

  // the wavefronts' results, column by column
  float* ml = smem + (size_t)W * max_cols * LD;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] = column_sum(l[ct]);
    const int c = ct * 16 + c16;
    if (c >= cols) continue;
    float* o = smem + ((size_t)wave * max_cols + c) * LD + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(o + 16 * dt) = acc[ct][dt];
    if (g == 0) {
      ml[2 * (wave * max_cols + c)] = bad ? __builtin_nanf("") : m[ct];
      ml[2 * (wave * max_cols + c) + 1] = l[ct];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < cols * (DH / 4); i += W * 64) {
    const int c = i / (DH / 4), d = 4 * (i - c * (DH / 4));
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = ml[2 * (w * max_cols + c)];
      nan |= mw != mw;
      top = fmaxf(top, mw);
    }
    const float use = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[2 * (w * max_cols + c)] - use);
      sum = fmaf(ml[2 * (w * max_cols + c) + 1], f, sum);
      const f32x4 v = *reinterpret_cast<const f32x4*>(smem + ((size_t)w * max_cols + c) * LD + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], f, o[e]);
    }
    const int t = c / G;
    if (ranges == 1) {
      const float inv = nan ? __builtin_nanf("") : (sum > 0.f ? 1.0f / sum : 0.f);
      *reinterpret_cast<u32x2*>(out + ((size_t)(n0 + t) * Hq + hk * G + c - t * G) * DH + d) =
          u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
    } else {
      const size_t slot = (((size_t)tile * Hkv + hk) * ranges + rng) * max_cols + c;
      *reinterpret_cast<f32x4*>(ws_o + slot * DH + d) = o;
      if (d == 0) {
        ws_ml[2 * slot] = nan ? __builtin_nanf("") : top;
        ws_ml[2 * slot + 1] = sum;
      }
    }
  }
}

// The ranges' results of every (tile, kv head, column), added up in the ranges' order: a wavefront each.
__global__ __launch_bounds__(256) void attention_quantized_merge_kernel(
    const float* __restrict__ ws_ml, const float* __restrict__ ws_o, bf16_t* __restrict__ out,
    const int* __restrict__ positions, const int* __restrict__ tiles, int num_tiles, int ranges, int range, int ret_mode,
    int ret_param, int Hq, int Hkv, int DH, int max_cols) {
  const int lane = threadIdx.x & 63;
  const int item = blockIdx.x * 4 + wave_index();
  if (item >= num_tiles * Hkv * max_cols) return;
  const int c = item % max_cols, hk = item / max_cols % Hkv, tile = item / (max_cols * Hkv);
  const int n0 = tiles[2 * tile], nt = tiles[2 * tile + 1];
  const int G = Hq / Hkv;
  if (c >= nt * G) return;
  const int p_first = positions[n0];
  const int first = first_key(ret_mode, ret_param, p_first);
  const int ns = (p_first + nt - 1) / range - first / range + 1;
  const size_t slot0 = ((size_t)tile * Hkv + hk) * ranges * max_cols + c;
  float top = -INFINITY;
  bool nan = false;
  for (int r = lane; r < ns; r += 64) {
    const float mr = ws_ml[2 * (slot0 + (size_t)r * max_cols)];
    nan |= mr != mr;
    top = fmaxf(top, mr);
  }
  top = wave_max(top);
  nan = __any(nan);
  const float use = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int r = lane; r < ns; r += 64)
    sum = fmaf(ws_ml[2 * (slot0 + (size_t)r * max_cols) + 1],
               __builtin_amdgcn_exp2f(ws_ml[2 * (slot0 + (size_t)r * max_cols)] - use), sum);
  sum = wave_sum(sum);
  const float inv = nan ? __builtin_nanf("") : (sum > 0.f ? 1.0f / sum : 0.f);
  const int t = c / G;
  bf16_t* dst = out + ((size_t)(n0 + t) * Hq + hk * G + c - t * G) * DH;
  for (int d = 4 * lane; d < DH; d += 256) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int r = 0; r < ns; ++r) {
      const float f = __builtin_amdgcn_exp2f(ws_ml[2 * (slot0 + (size_t)r * max_cols)] - use);
      const f32x4 v = *reinterpret_cast<const f32x4*>(ws_o + (slot0 + (size_t)r * max_cols) * DH + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], f, o[e]);
    }
    *reinterpret_cast<u32x2*>(dst + d) = u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
  }
}

// tiles: [num_tiles][2] = (first row, tokens), tokens * Hq / Hkv <= max_cols <= 64 (32 for heads of 256); every tile's
// tokens are consecutive positions of one segment.  ranges: the most ranges of `range` positions (a multiple of 32) that a
// tile reads.  ws_ml: [num_tiles][Hkv][ranges][max_cols][2], ws_o: the same with [dh]; null with one range.
JLE_API int jle_attention_quantized(const void* q, const void* codes, const void* scales, void* out, float* ws_ml,
                                    float* ws_o, const int* positions, const int* token_segment, const int* block_table,
                                    int table_width, int num_pages, const int* tiles, int num_tiles, int max_cols,
                                    int ranges, int range, int ret_mode, int ret_param, float scale, int Hq, int Hkv,
                                    int dh, int ps, hipStream_t s) {
  if (num_tiles <= 0) return 0;
  if (!quantized_head_ok(dh) || Hkv <= 0 || Hq % Hkv || ps < 16 || ps % 16 || max_cols < Hq / Hkv) return JLE_BAD_ARG;
  if (max_cols > (dh == 256 ? 32 : 64) || ranges < 1 || range < 32 || range % 32 || num_pages <= 0) return JLE_BAD_ARG;
  if (ranges > 1 && (ws_ml == nullptr || ws_o == nullptr)) return JLE_BAD_ARG;
  if ((ret_mode == 1 || ret_mode == 2) && ret_param <= 0) return JLE_BAD_ARG;
  if (!(scale > 0.f) || (((uintptr_t)q | (uintptr_t)codes | (uintptr_t)scales | (uintptr_t)out) & 15)) return JLE_BAD_ARG;
  const long long blocks = (long long)num_tiles * Hkv * ranges;
  if (blocks > (1ll << 30)) return JLE_BAD_ARG;
  const float sl = scale * kLog2e;
#define LAUNCH(DH, CT, W)                                                                                                   \
  do {                                                                                                                      \
    const size_t lds = (size_t)(W) * max_cols * ((DH) + 4 + 2) * sizeof(float);                                             \
    const int rc = allow_lds(attention_quantized_kernel<DH, CT, W>, lds);                                                   \
    if (rc) return rc;                                                                                                      \
    hipLaunchKernelGGL((attention_quantized_kernel<DH, CT, W>), dim3((unsigned)blocks), dim3((W) * 64), lds, s,             \
                       (const bf16_t*)q, (const uint8_t*)codes, (const uint8_t*)scales, (bf16_t*)out, ws_ml, ws_o,          \
                       positions, token_segment, block_table, table_width, num_pages, tiles, ranges, range, ret_mode,       \
                       ret_param, sl, Hq, Hkv, ps, max_cols);                                                               \
  } while (0)
#define PICK(DH)                               \
  do {                                         \
    if (max_cols <= 16) LAUNCH(DH, 1, 8);      \
    else if (max_cols <= 32) LAUNCH(DH, 2, 8); \
    else LAUNCH(DH, 4, 4);                     \
  } while (0)
  switch (dh) {
    case 32: PICK(32); break;
    case 64: PICK(64); break;
    case 96: PICK(96); break;
    case 128: PICK(128); break;
    case 256:
      if (max_cols <= 16) LAUNCH(256, 1, 4);
      else LAUNCH(256, 2, 4);
      break;
  }
#undef PICK
#undef LAUNCH
  JLE_LAUNCH_CHECK();
  if (ranges > 1) {
    const long long items = (long long)num_tiles * Hkv * max_cols;
    if (items > (1ll << 30)) return JLE_BAD_ARG;
    hipLaunchKernelGGL(attention_quantized_merge_kernel, dim3((unsigned)((items + 3) / 4)), dim3(256), 0, s, ws_ml, ws_o,
                       (bf16_t*)out, positions, tiles, num_tiles, ranges, range, ret_mode, ret_param, Hq, Hkv, dh, max_cols);
    JLE_LAUNCH_CHECK();
  }
  return 0;
}
