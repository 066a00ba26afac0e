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
// The softmax is one pass: a running maximum and sum a column, the accumulators rescaled where the maximum grows; scores,
// sums and accumulators are float32.  The probabilities times the scales are rounded to bfloat16 (half a step: 2^-8 of each),
// as they are where pages are bfloat16: the matrix instruction multiplies them by codes that it takes exactly.
//
// The pages hold the codes in the lanes' order, so every load of a wavefront is a contiguous kilobyte.  A wavefront holds one
// step of 32 keys and asks for the next one's keys and values as it is done with this one's: 118 registers at dh 128, two
// blocks of eight wavefronts a compute unit.  (Two steps in registers, one block a compute unit: 98 keys 4.7 us, not 4.0, eight
// requests of 2,100 13.3, not 11.8; steps of 64 keys, three steps on their way and sixteen wavefronts a block: no faster.)
// Where the launch fills the GPU memory bounds it, 2 * dh + 2 bytes a key and kv head: 64 requests of 6,100 keys on 8 kv heads
// of 128 133 us, 6.0 TB/s, 128 of 2,048 83 us, 6.5.  Where it does not, a wavefront's instructions do: about 300 a step, 1.2 us
// with two wavefronts a SIMD; hence blocks of eight wavefronts, and ranges: 32,768 keys of one request 18.5 us (13 at a copy's
// rate).
//
// The wavefronts' (maximum, sum, unnormalised O^T) are merged in shared memory; with more than one range a (tile, kv head)
// the blocks' results go through memory, and the block that takes the last ticket adds them up in the ranges' order.  Which
// ranges there are depends on the position, the retention rule and `range` alone.
#include "mfma_attention.h"
#include "quantized.h"

using namespace jle;

// The first key that a query at `pos` reads: rules all (0), chunk (1), window (2).
struct Rule {
  int mode;
  Divisor param;
  __device__ __forceinline__ int first(int pos) const {
    if (mode == 0) return 0;
    if (mode == 1) return over(pos, param) * (int)param.d;
    return max(pos - (int)param.d + 1, 0);
  }
};

template <int DH>
struct QuantizedStep {  // 32 keys of one kv head: two tiles of sixteen
  static constexpr int P = DH / 64;                // pieces of 64 elements
  static constexpr bool T = DH % 64 != 0;          // a last piece of 32
  u32x4 k[2][P > 0 ? P : 1], v[2][P > 0 ? P : 1];
  u32x2 kt[2], vt[2];
  uint32_t ks[2], vs[2];  // scale bytes: of the lane's key; of its four keys
};

__device__ __forceinline__ uint32_t two_codes(uint32_t w, float scale, bool hi) {
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
__device__ __forceinline__ bf16x8 eight_codes(uint32_t a, uint32_t b, float scale) {
  const u32x4 r = {two_codes(a, scale, false), two_codes(a, scale, true), two_codes(b, scale, false), two_codes(b, scale, true)};
  return __builtin_bit_cast(bf16x8, r);
}

// Two floats written to / read from where all compute units see them at once: for what blocks on different dies hand each
// other within a launch.
typedef __attribute__((ext_vector_type(2))) float f32x2;
__device__ __forceinline__ void put_through(float* p, float a, float b) {
  const f32x2 v = {a, b};
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 get_through(const float* p) {
  return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                     __HIP_MEMORY_SCOPE_AGENT));
}
constexpr int kMostRanges = 64;  // of a (tile, kv head): their maxima and sums fit where the wavefronts' results lay

static_assert(kMostRanges * sizeof(f32x2) <= 4 * (32 + 4) * sizeof(float), "a column's maxima and sums in its results' place");

// (up to 16 columns and dh 128: two blocks a compute unit; otherwise one)
template <int DH, int CT, int W>
__global__ __launch_bounds__(W * 64, CT == 1 && DH <= 128 ? 4 : W / 4) void attention_quantized_kernel(
    const bf16_t* q, const uint8_t* codes, const uint8_t* scales,
    bf16_t* __restrict__ out, float* __restrict__ ws_ml, float* __restrict__ ws_o, int* __restrict__ tickets,
    const int* __restrict__ positions, const int* __restrict__ token_segment, const int* __restrict__ block_table,
    int table_width, int num_pages, const int* __restrict__ tiles, int ranges, Divisor range, Rule rule, float scale_log2, int Hq, int Hkv, Divisor group,
    Divisor page_tiles, int max_cols) {
  using Step = QuantizedStep<DH>;
  constexpr int P = Step::P, DT = DH / 16, KC = DH / 32, LD = DH + 4;
  extern __shared__ __attribute__((aligned(16))) float smem[];  // [W][max_cols][LD], then [W][max_cols][2]
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int c16 = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x, tile = blockIdx.y, rng = blockIdx.z;  // (ranges that few tiles have come last)
  const int ps = 16 * (int)page_tiles.d, G = (int)group.d;
  const int n0 = tiles != nullptr ? tiles[2 * tile] : tile, nt = tiles != nullptr ? tiles[2 * tile + 1] : 1;
  const int p_first = positions[n0], p_last = p_first + nt - 1;
  if (p_last < 0) {  // rows at no position (a batch filled up with such) see no keys: nothing of theirs is looked up
    for (int i = threadIdx.x; rng == 0 && i < nt * G * (DH / 4); i += W * 64) {
      const int c = i / (DH / 4), t = over(c, group);
      *reinterpret_cast<u32x2*>(out + ((size_t)(n0 + t) * Hq + hk * G + c - t * G) * DH + 4 * (i - c * (DH / 4))) = u32x2{0u, 0u};
    }
    return;
  }
  const int first = rule.first(max(p_first, 0));
  const int r_first = over(first, range), r_abs = r_first + rng;
  const int all_ranges = over(p_last, range) - r_first + 1, mine = min(all_ranges, ranges);
  if (rng >= mine) return;  // (this tile has fewer ranges)
  const int k_lo = max(first, r_abs * (int)range.d), k_hi = min(p_last, r_abs * (int)range.d + (int)range.d - 1);
  const int full_lo = max(k_lo, rule.first(p_last)), full_hi = min(k_hi, p_first);
  const int cols = nt * G;
  const int* table = block_table + (size_t)token_segment[n0] * table_width;

  float m[CT], l[CT];
  f32x4 acc[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bool bad = all_ranges > ranges;  // (keys beyond what the launch was laid out for: the result is NaN)
  int lo[CT], hi[CT];
  bf16x8 qb[CT][KC];

  // The keys of a wavefront's next step are asked for when this step's scores are formed, its values when this step's are added
  // up: one step's registers, and the loads of both on their way meanwhile.  Their pages are looked up, through the scalar
  // path, a step before that: no load waits for the block table.  And every load in the loop is issued, whether its keys exist
  // or not (then it reads the range's nearest tile, and what it brings is masked): the waits count loads, and no way through the
  // loop may leave one out.  A wavefront's last step asks for nothing and stands behind the loop (98 keys 4.2 -> 4.0 us).
  struct Pages {
    int id[2], off[2];  // per tile of sixteen keys: its page, the place of its first key there
  };
  const int tile_lo = k_lo >> 4, tile_hi = k_hi >> 4;
  bad |= over(tile_hi, page_tiles) >= table_width;
  auto look_up = [&](Pages& at, int step) {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int kt = min(max(2 * step + tt, tile_lo), tile_hi), idx = over(kt, page_tiles);
      at.id[tt] = table[min(idx, table_width - 1)];
      at.off[tt] = 16 * (kt - idx * (int)page_tiles.d);
    }
  };
  const uint32_t page_rows = (uint32_t)Hkv * 2 * ps;
  auto row_of = [&](const Pages& at, int tt) {  // of the tile's first key, among all pages' keys and values
    const bool ok = (uint32_t)at.id[tt] < (uint32_t)num_pages;
    bad |= !ok;  // (a page is missing: the result is NaN)
    return (uint64_t)(uint32_t)(ok ? at.id[tt] : 0) * page_rows + (uint32_t)(hk * 2 * ps + at.off[tt]);
  };
  Step s;
  auto load_keys = [&](const Pages& at) {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const uint64_t row = row_of(at, tt);
      const uint8_t* kp = codes + row * DH;
      s.ks[tt] = scales[row + c16];
#pragma unroll
      for (int p = 0; p < P; ++p) s.k[tt][p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + 1024 * p) + lane);
      if (Step::T) s.kt[tt] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(kp + 1024 * P) + lane);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto load_values = [&](const Pages& at) {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const uint64_t row = row_of(at, tt) + ps;
      const uint8_t* vp = codes + row * DH;
      s.vs[tt] = *reinterpret_cast<const uint32_t*>(scales + row + 4 * g);
#pragma unroll
      for (int p = 0; p < P; ++p) s.v[tt][p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp + 1024 * p) + lane);
      if (Step::T) s.vt[tt] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vp + 1024 * P) + lane);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  auto work = [&](auto more, int step, const Pages& next) {
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
    __builtin_amdgcn_sched_barrier(0);
    if (more.value) load_keys(next);
    const bool full = 32 * step >= full_lo && 32 * step + 31 <= full_hi;
    if (!full) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        // Values and scales of keys outside the range may never have been written: they are read as zero.  So is a row that is
        // NaN throughout: some columns may not see its key, and those that do have NaN from its score.
        const uint32_t none = codes_none(P > 0 ? s.v[tt][0][0] : s.vt[tt][0]);
        uint32_t keep = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = 32 * step + 16 * tt + 4 * g + i;
          const bool nan = none >> (8 * i) & 1u;
          keep |= (key >= k_lo) & (key <= k_hi) & !nan ? 255u << (8 * i) : 0u;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            const float seen = nan ? __builtin_nanf("") : st[ct][tt][i];
            st[ct][tt][i] = (key >= lo[ct]) & (key <= hi[ct]) ? seen : -INFINITY;
          }
        }
        s.vs[tt] &= keep;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int j = 0; j < 4; ++j) s.v[tt][p][j] &= keep;
        if (Step::T) {
          s.vt[tt][0] &= keep;
          s.vt[tt][1] &= keep;
        }
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
      const bf16x8 a = eight_codes(tail ? s.vt[0][dt & 1] : s.v[0][dt / 4][dt & 3],
                                   tail ? s.vt[1][dt & 1] : s.v[1][dt / 4][dt & 3], 1.0f);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[ct], acc[ct][dt], 0, 0, 0);
    }
  };

  const int last = k_hi / 32;
  int step = k_lo / 32 + wave;
  Pages next, after;
  look_up(next, step);
  look_up(after, step + W);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = ct * 16 + c16;
    const int t = c < cols ? over(c, group) : 0, head = hk * G + (c < cols ? c - t * G : 0);
    lo[ct] = max(k_lo, rule.first(p_first + t));
    hi[ct] = min(k_hi, p_first + t);
    const bf16_t* row = q + ((size_t)(n0 + t) * Hq + head) * DH;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      qb[ct][2 * p] = *reinterpret_cast<const bf16x8*>(row + 64 * p + 16 * g);
      qb[ct][2 * p + 1] = *reinterpret_cast<const bf16x8*>(row + 64 * p + 16 * g + 8);
    }
    if (Step::T) qb[ct][KC - 1] = *reinterpret_cast<const bf16x8*>(row + 64 * P + 8 * g);
  }
  __builtin_amdgcn_sched_barrier(0);  // (the queries first: the loop's waits count what is asked for behind them)
  load_keys(next);
  load_values(next);
  for (; step + W <= last; step += W) {
    next = after;
    look_up(after, step + 2 * W);
    work(std::true_type(), step, next);
    load_values(next);
  }
  if (step <= last) work(std::false_type(), step, next);
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
  // (column, four elements) items: a block's result, or its part of one
  const size_t part0 = ((size_t)tile * Hkv + hk) * ranges;
  const bool alone = mine == 1;
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
    if (alone) {
      const int t = over(c, group);
      const float inv = nan ? __builtin_nanf("") : (sum > 0.f ? 1.0f / sum : 0.f);
      *reinterpret_cast<u32x2*>(out + ((size_t)(n0 + t) * Hq + hk * G + c - t * G) * DH + d) =
          u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
    } else {
      const size_t slot = (part0 + rng) * max_cols + c;
      put_through(ws_o + slot * DH + d, o[0], o[1]);
      put_through(ws_o + slot * DH + d + 2, o[2], o[3]);
      if (d == 0) put_through(ws_ml + 2 * slot, nan ? __builtin_nanf("") : top, sum);
    }
  }
  if (alone) return;

  // Every wavefront waits until its stores have got to where all compute units read them (vmcnt(0)), then the barrier, then
  // one thread takes a ticket, atomically for the whole GPU: whoever takes the last one knows that all parts are there, and
  // reads them past its own die's caches.  It puts the counter back to zero for the next launch.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __syncthreads();  // (also: nobody reads ml any more)
  int* last_flag = reinterpret_cast<int*>(ml);
  if (threadIdx.x == 0) {
    int* ticket = tickets + (size_t)tile * Hkv + hk;
    const bool is_last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == mine - 1;
    if (is_last) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *last_flag = is_last;
  }
  __syncthreads();
  if (!*last_flag) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  f32x2* parts = reinterpret_cast<f32x2*>(smem);  // [mine][cols]: the parts' maxima and sums
  for (int i = threadIdx.x; i < mine * cols; i += W * 64) {
    const int r = i / cols, c = i - r * cols;
    parts[i] = get_through(ws_ml + 2 * ((part0 + r) * max_cols + c));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < cols * (DH / 2); i += W * 64) {
    const int c = i / (DH / 2), d = 2 * (i - c * (DH / 2));
    const float* po = ws_o + (part0 * max_cols + c) * DH + d;
    float top = -INFINITY, sum = 0.f;
    bool nan = false;
    for (int r = 0; r < mine; ++r) {
      const float mr = parts[r * cols + c][0];
      nan |= mr != mr;
      top = fmaxf(top, mr);
    }
    const float use = top == -INFINITY ? 0.f : top;
    f32x2 o = {0.f, 0.f};
    for (int r0 = 0; r0 < mine; r0 += 8) {  // eight parts' numbers on their way at once, added up in the ranges' order
      f32x2 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = get_through(po + (size_t)min(r0 + k, mine - 1) * max_cols * DH);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const f32x2 part = parts[min(r0 + k, mine - 1) * cols + c];
        const float f = r0 + k < mine ? __builtin_amdgcn_exp2f(part[0] - use) : 0.f;
        sum = fmaf(part[1], f, sum);
        o[0] = fmaf(v[k][0], f, o[0]);
        o[1] = fmaf(v[k][1], f, o[1]);
      }
    }
    const float inv = nan ? __builtin_nanf("") : (sum > 0.f ? 1.0f / sum : 0.f);
    const int t = over(c, group);
    *reinterpret_cast<uint32_t*>(out + ((size_t)(n0 + t) * Hq + hk * G + c - t * G) * DH + d) = pack_bf16(o[0] * inv, o[1] * inv);
  }
}

// tiles: [num_tiles][2] = (first row, tokens), tokens * Hq / Hkv <= max_cols <= 32; every tile's
// tokens are consecutive positions of one segment.  ranges: the most ranges of `range` positions (a multiple of 32) that a
// tile reads.  ws_ml: [num_tiles][Hkv][ranges][max_cols][2], ws_o: the same with [dh], tickets: [num_tiles][Hkv], zero before
// and after; null with one range.  tiles null: tile i is the single token i.  More tiles than kMostTiles: several launches.
constexpr int kMostTiles = 65535;  // of a launch: the grid's second dimension
JLE_API int jle_attention_quantized(const void* q, const void* codes, const void* scales, void* out, float* ws_ml,
                                    float* ws_o, int* tickets, const int* positions, const int* token_segment, const int* block_table,
                                    int table_width, int num_pages, const int* tiles, int num_tiles, int max_cols,
                                    int ranges, int range, int ret_mode, int ret_param, float scale, int Hq, int Hkv,
                                    int dh, int ps, hipStream_t s) {
  if (num_tiles <= 0) return 0;
  if (!quantized_head_ok(dh) || Hkv <= 0 || Hq % Hkv || ps < 16 || ps % 16 || max_cols < Hq / Hkv) return JLE_BAD_ARG;
  if (table_width < 1 || max_cols > 32 || ranges < 1 || range < 32 || range % 32 || num_pages <= 0) return JLE_BAD_ARG;
  if (ranges > 1 && (ws_ml == nullptr || ws_o == nullptr || tickets == nullptr)) return JLE_BAD_ARG;
  if ((ret_mode == 1 || ret_mode == 2) && ret_param <= 0) return JLE_BAD_ARG;
  if (((uintptr_t)ws_ml | (uintptr_t)ws_o) & 7) return JLE_BAD_ARG;
  if (!(scale > 0.f) || (((uintptr_t)q | (uintptr_t)codes | (uintptr_t)scales | (uintptr_t)out) & 15)) return JLE_BAD_ARG;
  if (ranges > kMostRanges) return JLE_BAD_ARG;
  const float sl = scale * kLog2e;
  const Rule rule = {ret_mode, divisor(ret_mode == 0 ? 1 : ret_param)};
#define LAUNCH(DH, CT, W)                                                                                                   \
  do {                                                                                                                      \
    const size_t lds = (size_t)(W) * max_cols * ((DH) + 4 + 2) * sizeof(float);                                             \
    const int rc = lds > 64 * 1024 ? allow_lds(attention_quantized_kernel<DH, CT, W>, lds) : 0;                             \
    if (rc) return rc;                                                                                                      \
    hipLaunchKernelGGL((attention_quantized_kernel<DH, CT, W>), dim3(Hkv, num, ranges), dim3((W) * 64), lds, s,             \
                       (const bf16_t*)q + row * Hq * (DH), (const uint8_t*)codes, (const uint8_t*)scales,                   \
                       (bf16_t*)out + row * Hq * (DH), ws_ml + 2 * slot, ws_o + slot * (DH), tickets + counter,             \
                       positions + row, token_segment + row, block_table, table_width, num_pages,                           \
                       tiles == nullptr ? nullptr : tiles + 2 * (size_t)t0, ranges, divisor(range), rule, sl, Hq, Hkv,      \
                       divisor(Hq / Hkv), divisor(ps / 16), max_cols);                                                      \
  } while (0)
#define PICK(DH)                               \
  do {                                         \
    if (max_cols <= 16) LAUNCH(DH, 1, 8);      \
    else LAUNCH(DH, 2, (DH) <= 128 ? 8 : 4);   \
  } while (0)
  for (int t0 = 0, num; t0 < num_tiles; t0 += num) {
    num = num_tiles - t0 < kMostTiles ? num_tiles - t0 : kMostTiles;
    const size_t row = tiles == nullptr ? t0 : 0;  // (listed tiles name their rows among all)
    const size_t counter = ranges > 1 ? (size_t)t0 * Hkv : 0, slot = counter * ranges * max_cols;
    switch (dh) {
      case 32: PICK(32); break;
      case 64: PICK(64); break;
      case 96: PICK(96); break;
      case 128: PICK(128); break;
      case 256: PICK(256); break;
    }
  }
#undef PICK
#undef LAUNCH
  JLE_LAUNCH_CHECK();
  return 0;
}
