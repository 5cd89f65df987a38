// Differential attention: o_i = sum_j (P1 - lam P2)_ij v_j, P_m = softmax_j(scale q_m,i . k_m,j) over the keys that query i sees.
//
//   rows      the queries of one (sample, key head) and its G = heads / kv_heads query heads are packed into R = nq G rows, row r = query
//             r / G, head r % G of the group: a key tile is read once for all heads that share it, and the gradients of shared keys
//             are sums inside one workgroup (no atomics anywhere; every result has one fixed summation order).
//   visible   key j < end(i): end = len (no mask), min(len, i + 1) ("start") or len - nq + 1 + i ("end").  Keys at or behind len, or that no row
//             of the workgroup sees, are not multiplied (their rows are clamped to the last seen one, their scores replaced, and dK / dV replace the
//             products), so anything may stand there.  A value that a mask hides from one row and not from its neighbours has to be a number.
//             A row that sees nothing gives 0, lse = +inf, and no gradient.
//   waves     a wave works on 32 rows (or 32 keys) of ONE map; two neighbouring waves hold the two maps of the same rows and meet once at the end,
//             lane to lane through LDS.  That halves a wave's registers (one accumulator set, one resident operand), so that two to four
//             waves share a SIMD and hide each other's latencies.  The forward repeats nothing by it; the backward computes dP = dO V^T
//             and the product with dO once per map (dK / dV: 72 matrix instructions per 32 x 32 tile at d = 64 for 48) and is still far ahead:
//             with both maps in one wave, one wave per SIMD, dK / dV took 849 us for 535 at (2, 4096, 16 / 4 heads, 64 / 128, bf16, causal), P and
//             dS as one term.
//   forward   one pass over the keys: S^T = K Q^T (a lane owns one query), running maximum and sum in 32 bits, O^T += V^T P^T.
//             The maximum only moves when a score passes it by 2^8 (the weights stay <= 2^8, far inside every type), which makes
//             the rescaling of the accumulators rare.
//   backward  dP = dO V^T; D_m = dO . O_m; dS_1 = P1 (dP - D_1), dS_2 = -lam P2 (dP - D_2);
//             dQ_m = scale dS_m K_m, dK_m = scale dS_m^T Q_m, dV = (P1 - lam P2)^T dO, dlam = -sum D_2.  Scores are recomputed from lse.
//             dK / dV: a wave owns 32 keys and walks the rows; dQ: a wave owns 32 rows and walks the keys.
// Scores, sums, lse, D, the maps' own products that D is formed from and all accumulators are 32-bit; only results are rounded to the inputs' type.  P
// and dS are the left operands of 16-bit matrix instructions: they enter as two terms (mm_transposed), for any number of rows.  At (2, 4096, 16 / 4 heads,
// 64 / 128, bf16, causal) that is 1350 - 1430 us a training pass where one rounding took 1016, and results are as far from 64 bits as their own rounding is (0.0017
// of the norm in bf16, 0.0002 in fp16; one rounding: 0.0027, 0.0003); single tokens are bound by the cache's bytes and pay nothing.
#pragma once
#include "../../include/immunostruct_hip.h"
#include "tiles16.h"

namespace is {
namespace da {

typedef IsDiffAttention Args;
// The forward's weights are taken as 2^LIFT exp(score - running maximum), which may fall behind the true one by 2^SLACK.  fp16 has no steps below 2^-24:
// there the largest weight is kept at 2^8 ... 2^12, so that what is lost lies below 2^-33 of it (unlifted, 4000 keys of weight 2^-26 beside one of weight 1
// came out as nothing).  Four bits stay free above: the exponents are taken against a rounded maximum, which at scores of 10^7 and more is off by whole
// units.  The other types have fp32's range; the larger slack makes rescaling rarer.
template <typename T> constexpr float lift_of() { return __is_same(T, _Float16) ? 8.0f : 0.0f; }
template <typename T> constexpr float slack_of() { return __is_same(T, _Float16) ? 4.0f : 8.0f; }

typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int V> struct Int { static constexpr int value = V; };
// steps j0 = first, first + STEP ... below last, alternating between two buffers whose number is a compile-time constant
// (LDS addresses then are loop-invariant registers plus immediates)
template <int STEP, typename F>
__device__ __forceinline__ void two_buffers(int first, int last, F step) {
  for (int j0 = first; j0 < last; j0 += 2 * STEP) {
    step(j0, Int<0>());
    if (j0 + STEP < last) step(j0 + STEP, Int<1>());
  }
}

// Row (key) groups of a workgroup: two waves each.  More groups share a staged tile, fewer let the workgroups of a CU drift apart, so that one multiplies
// while another forms weights, and waste less on the last rows of short samples.  Measured (us) for 2 / 4 groups, where a build of 4 fits its registers and LDS:
//   width 32   fp32 (128, 190, 1 head, ragged): forward 30.1 / 31.9, dK / dV 49.2 / 50.9, dQ 31.8 / 33.0; bf16 (4, 1024, 8 / 4 heads, causal): 31 / 41,
//              46 / 56, 29 / 37; bf16 (128, 190, 2 heads, ragged): 19 / 23, 24 / 34, 14 / 16
//   width 64   bf16 (2, 4096, 16 / 4 heads, causal): 422 / 429, 725 / 688, 431 / 442; fp32 (1, 2048, 2 heads, causal): 59 / 67, - , 282 / 488; fp32 (16, 300,
//              4 / 2 heads, ragged): 77 / 74, - , 99 / 89
//   width 128  fp16 (5, 517 over 1531, 6 / 2 heads): 103 / 117, - , 109 / 110
// Two groups, then, but for the 16-bit dK / dV at width 64.
template <typename T, int D> constexpr int fwd_groups() { return 2; }
template <typename T, int D> constexpr int key_groups() { return sizeof(T) == 2 && D == 64 ? 4 : 2; }
template <typename T, int D> constexpr int dq_groups() { return 2; }

template <typename T>
__device__ __forceinline__ float lam_at(const Args& a, int head) {
  return a.lam_type == TYPE_F32 ? reinterpret_cast<const float*>(a.lam)[head] : (float)reinterpret_cast<const T*>(a.lam)[head];
}
__device__ __forceinline__ int length_of(const Args& a, int b) {
  const int n = a.lengths != nullptr ? a.lengths[b] : a.nk;
  return n < 0 ? 0 : (n > a.nk ? a.nk : n);
}
// keys [0, end) are visible to query i
__device__ __forceinline__ int end_of(const Args& a, int i, int len) {
  if (a.causal == 0) return len;
  const int e = a.causal == 1 ? i + 1 : len - a.nq + 1 + i;
  return e < 0 ? 0 : (e < len ? e : len);
}
// first query that sees key j (nq: none does)
__device__ __forceinline__ int first_query(const Args& a, int j, int len) {
  if (a.causal == 0) return 0;
  const int i = a.causal == 1 ? j : j - (len - a.nq);
  return i < 0 ? 0 : (i < a.nq ? i : a.nq);
}

// row r -> (query, head of the group): r / group by a 32-bit reciprocal (floor((2^32 - 1) / group)), at most one too small
__device__ __forceinline__ int query_of(const Args& a, int r, int& g) {
  int i = (int)__umulhi((unsigned)r, a.group_magic);
  g = r - i * a.group;
  if (g >= a.group) {
    ++i;
    g -= a.group;
  }
  return i;
}
// element (b, query i, head h) of a contiguous (batch, nq, heads, dv) tensor
__device__ __forceinline__ long long o_at(const Args& a, int b, int i, int h) { return (((long long)b * a.nq + i) * a.heads + h) * a.dv; }
// elements of one map's product in `maps` (2, batch, nq, heads, dv)
__device__ __forceinline__ long long maps_plane(const Args& a) { return (long long)a.batch * a.nq * a.heads * a.dv; }

// The two maps' rows of a tile lie behind each other: tile rows [0, n) are map 0's, [n, 2 n) map 1's (MAPS = 2; 1: values, one set).
// byte offsets of a tile's key rows, clamped to the last valid one, from its first row
template <typename S, int MAPS>
__device__ __forceinline__ void key_offsets(unsigned (&out)[S::PER], int tid, unsigned stride, unsigned map, int left) {
  constexpr int N = S::ROWS_ / MAPS;
#pragma unroll
  for (int k = 0; k < S::PER; ++k) {
    const int row = S::row_of(tid, k);
    out[k] = (unsigned)min(row & (N - 1), left) * stride + (row >= N ? map : 0u);
  }
}
// byte offsets of a tile's packed rows, clamped to the last one, from query r0 / group and the group's first head
template <typename S, int MAPS>
__device__ __forceinline__ void row_offsets(const Args& a, unsigned (&out)[S::PER], int tid, int r0, int first, unsigned stride, unsigned head, unsigned map) {
  constexpr int N = S::ROWS_ / MAPS;
#pragma unroll
  for (int k = 0; k < S::PER; ++k) {
    const int row = S::row_of(tid, k);
    int g;
    const int i = query_of(a, min(r0 + (row & (N - 1)), a.rows - 1), g);
    out[k] = (unsigned)(i - first) * stride + (unsigned)g * head + (row >= N ? map : 0u);
  }
}
// Hands the wave of map 1's accumulators to the wave of map 0 of the same rows: f(t, own, other) runs in map 0's lanes with both values of
// 32-column block t (f32x16 each).  `lds`: BYTES of scratch; every wave of the workgroup takes part.
template <int NT, int GROUPS, int BYTES, typename F>
__device__ __forceinline__ void hand_over(const f32x16 (&acc)[NT], char* lds, int group, int map, int lane, F f) {
  constexpr int FIT = BYTES / (GROUPS * 4096), STEP = FIT < NT ? FIT : NT;
  static_assert(STEP >= 1, "one block of every group has to fit");
  f32x4* mine = reinterpret_cast<f32x4*>(lds) + group * 256 + lane;
#pragma unroll
  for (int t0 = 0; t0 < NT; t0 += STEP) {
    __syncthreads();
    if (map == 1) {
#pragma unroll
      for (int t = t0; t < t0 + STEP && t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 4; ++u) mine[(t - t0) * GROUPS * 256 + u * 64] = f32x4{acc[t][4 * u], acc[t][4 * u + 1], acc[t][4 * u + 2], acc[t][4 * u + 3]};
    }
    __syncthreads();
    if (map == 0) {
#pragma unroll
      for (int t = t0; t < t0 + STEP && t < NT; ++t) {
        f32x16 other;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 x = mine[(t - t0) * GROUPS * 256 + u * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) other[4 * u + e] = x[e];
        }
        f(t, acc[t], other);
      }
    }
  }
}

// Keeps the left operands of a sum of products inside fp16's range: x is multiplied by a power of two of the lane's column, chosen at the first values and
// lowered (with the sums so far) only when one passes 2^15; values below 2^-34 of a column's largest are lost.  Score gradients are P dO V: over thousands of
// keys, or of small upstream gradients, they lie far below fp16's steps while the sums they belong to do not (dO of 1e-4 over 4096 keys: dQ was off by 6 x
// what rounding it costs), and large ones pass its largest number.  The other types have fp32's range and take x as it is.
template <typename T>
struct ColumnScale {
  static constexpr bool USED = __is_same(T, _Float16);
  float factor = USED ? 0x1p60f : 1.0f;
  template <int NT>
  __device__ __forceinline__ void fit(f32x16& x, f32x16 (&acc)[NT]) {
    if constexpr (USED) {
      float high = fabsf(x[0]);
#pragma unroll
      for (int t = 1; t < 16; ++t) high = fmaxf(high, fabsf(x[t]));
      if (__any(high * factor > 0x1p15f)) {
        const float most = fmaxf(high, other_half(high));      // (both halves of a wave hold rows of the same 32 columns)
        const float now = most * factor > 0x1p15f ? __builtin_ldexpf(1.0f, 10 - __builtin_amdgcn_frexp_expf(most)) : factor;
        const float shrink = now / factor;
        factor = now;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[t][e] *= shrink;
      }
#pragma unroll
      for (int t = 0; t < 16; ++t) x[t] *= factor;
    }
  }
};

// ---- forward -----------------------------------------------------------------------------------------------------------------------
// grid: (row tiles x splits x kv_heads x batch), GROUPS x 2 waves of 32 rows and one map.  splits > 1: every workgroup takes one range of the
// keys and leaves unnormalised sums with their maxima in the workspace; join_kernel puts them together.
// Bound by matrix instructions and the exponentials between them: (2, 4096, 16 / 4 heads, 64 / 128, bf16, "start") 430 us = 0.80 PFLOP/s executed
// (the product with V once per map and term; a large library product reaches 1.18); (5, 517 x 1531, 6 / 2, 128 / 256, fp16) 103 us, where the two-wave cap
// of 256 registers makes 128-wide heads spill 28 - 40 of them to scratch; (128, 190, 1, 32 / 64, fp32) 29 us, where fp32 matrix instructions
// share the vector pipe.  Single tokens are bound by the cache: (16, 1 x 16384 ragged, 16 / 4, 64 / 128, bf16) 77 us = 4.7 TB/s.
template <typename T, int D, int GROUPS, bool VEC>
__global__ __launch_bounds__(128 * GROUPS) __attribute__((amdgpu_waves_per_eu(2))) void fwd_kernel(const Args a) {
  constexpr int DV = 2 * D, KT = 32, NT = DV / 32, NJ = D / (2 * Vec<T>::N), NTH = 128 * GROUPS, SZ = sizeof(T);
  constexpr int KB = Tile<T, D>::bytes(KT), VB = Tile<T, DV>::bytes(KT), BUF = 2 * KB + VB;
  __shared__ __align__(16) char lds[2 * BUF];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 31, g = lane >> 5;
  const int group = wave >> 1, map = wave & 1;
  const int R = a.rows, tiles = (R + 32 * GROUPS - 1) / (32 * GROUPS);
  int base, unit;
  grid_order(blockIdx.x, a.batch * a.kv_heads, tiles * a.splits, base, unit);
  const int split = unit % a.splits, tile = tiles - 1 - unit / a.splits;      // the rows that see most keys first
  const int b = base / a.kv_heads, hk = base - b * a.kv_heads;
  const int len = length_of(a, b);
  const int row0 = (tile * GROUPS + group) * 32, r = row0 + qi, rr = r < R ? r : R - 1;
  int gi;
  const int query = query_of(a, rr, gi), head = hk * a.group + gi;
  const int wg_end = end_of(a, (min((tile + 1) * GROUPS * 32, R) - 1) / a.group, len);
  const int my_end = r < R ? end_of(a, query, len) : 0;
  const int wave_end = row0 < R ? end_of(a, min(row0 + 31, R - 1) / a.group, len) : 0;      // no row of the wave sees further
  const int wave_all = row0 + 31 < R ? end_of(a, row0 / a.group, len) : 0;                  // every row of the wave sees this far
  const int per = ((wg_end + a.splits - 1) / a.splits + KT - 1) / KT * KT;
  const int first = split * per, last = min(wg_end, first + per);
  const float c = a.scale * 1.44269504088896340736f;
  constexpr float LIFT = lift_of<T>(), SLACK = slack_of<T>();

  u32x4_t q[NJ];
  const char* qp = reinterpret_cast<const char*>(a.q) + (b * a.q_b + query * a.q_n + (2 * head + map) * a.q_h) * SZ;
#pragma unroll
  for (int j = 0; j < NJ; ++j) q[j] = load_chunk<T, VEC>(qp, 2 * j + g, a.d);
  const int k_at = map * KB + Tile<T, D>::rows_at(lane), v_at = 2 * KB + Tile<T, DV>::columns_at(lane);
  f32x16 o[NT];
  zero_acc(o);
  float top = -INFINITY, ref = 0.0f, sum = 0.0f;      // ref: what the exponents are taken against (LIFT - top c; 0 before the first key)

  typedef Stage<T, D, 2 * KT, NTH, VEC> StageK;
  typedef Stage<T, DV, KT, NTH, VEC> StageV;
  StageK sk;
  StageV sv;
  const char* kp = reinterpret_cast<const char*>(a.k) + (b * a.k_b + 2 * hk * a.k_h) * SZ;
  const char* vp = reinterpret_cast<const char*>(a.v) + (b * a.v_b + hk * a.v_h) * SZ;
  auto fetch = [&](int j0) {
    unsigned ko[StageK::PER], vo[StageV::PER];
    key_offsets<StageK, 2>(ko, tid, (unsigned)a.k_n * SZ, (unsigned)a.k_h * SZ, wg_end - 1 - j0);
    key_offsets<StageV, 1>(vo, tid, (unsigned)a.v_n * SZ, 0, wg_end - 1 - j0);
    sk.load(tid, kp + j0 * a.k_n * SZ, ko, a.d);
    sv.load(tid, vp + j0 * a.v_n * SZ, vo, a.dv);
  };
  auto place = [&](char* buf) {
    sk.store(tid, buf, a.d);
    sv.store(tid, buf + 2 * KB, a.dv);
  };
  if (first < last) {      // (uniform over the workgroup, as is every barrier below)
    fetch(first);
    place(lds);
    __syncthreads();
    two_buffers<KT>(first, last, [&](int j0, auto which) {
      constexpr int CUR = decltype(which)::value;
      const char* buf = lds + CUR * BUF;
      const bool more = j0 + KT < last;
      if (more) fetch(j0 + KT);
      if (j0 < wave_end) {
        f32x16 p = mm_tile<T, D>(buf + k_at, q);
        if (j0 + KT > wave_all) {
#pragma unroll
          for (int t = 0; t < 16; ++t) p[t] = j0 + tile_row(t, g) >= my_end ? -INFINITY : p[t];
        }
        float high = p[0];
#pragma unroll
        for (int t = 1; t < 16; ++t) high = fmaxf(high, p[t]);
        if (__any((high - top) * c > SLACK)) {
          const float now = fmaxf(top, fmaxf(high, other_half(high)));
          const float shrink = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((top - now) * c);
          top = now;
          ref = now == -INFINITY ? 0.0f : LIFT - now * c;
          sum *= shrink;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[t][e] *= shrink;
        }
        float add = 0.0f;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          p[t] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[t], c, ref));
          add += p[t];
        }
        sum += add;
        mm_transposed<T, DV, NT>(o, buf + v_at, p);
      }
      if (more) {
        place(lds + (CUR ^ 1) * BUF);
        __syncthreads();
      }
    });
  }
  const float total = sum + other_half(sum);
  const bool live = r < R;
  if (a.splits > 1) {
    if (!live) return;
    float* w = a.work + (((long long)base * a.splits + split) * 2 + map) * ((long long)R * (a.dv + 2)) + (long long)r * (a.dv + 2);
    if (g == 0) {
      w[a.dv] = top == -INFINITY ? -INFINITY : top * c - LIFT;
      w[a.dv + 1] = total;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        store4<float, false>(w, 32 * t + 8 * u + 4 * g, a.dv, f32x4{o[t][4 * u], o[t][4 * u + 1], o[t][4 * u + 2], o[t][4 * u + 3]});
    return;
  }
  const float inv = total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[t][e] *= inv;
  if (a.lse != nullptr && live && g == 0) a.lse[((long long)base * 2 + map) * R + r] = total != 0.0f ? __builtin_fmaf(top, c, __log2f(total)) - LIFT : INFINITY;
  const long long at = o_at(a, b, query, head);
  if (a.maps != nullptr && live) {
    float* mine = a.maps + map * maps_plane(a) + at;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        store4<float, VEC>(mine, 32 * t + 8 * u + 4 * g, a.dv, f32x4{o[t][4 * u], o[t][4 * u + 1], o[t][4 * u + 2], o[t][4 * u + 3]});
  }
  const float lam = lam_at<T>(a, head);
  T* out = reinterpret_cast<T*>(a.o) + at;
  hand_over<NT, GROUPS, 2 * BUF>(o, lds, group, map, lane, [&](int t, const f32x16& x, const f32x16& y) {
    if (!live) return;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 z;
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = x[4 * u + e] - lam * y[4 * u + e];
      store4<T, VEC>(out, 32 * t + 8 * u + 4 * g, a.dv, z);
    }
  });
}

__device__ __forceinline__ float wave_max(float v) {
  v = max_over_r(v);
  return fmaxf(v, other_half(v));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = sum_over_r(v);
  return v + other_half(v);
}

// The splits of one row put together by WAVES waves.  lane = split for the maxima and sums (at most 64 splits; every wave forms the weights), then
// a wave takes every WAVES-th split and a lane two columns: the first sums are loaded before their weights are known.  Single tokens have
// few rows and many splits: four waves a row (a workgroup), 4.8 us for 256 rows of 16 splits, 12.4 by one.  More rows: one, 7 us less than by four at
// (1, 512 over 4096, 8 / 2 heads, 64) bf16.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  constexpr int BATCH = 4;
  __shared__ __align__(16) f32x4 part[4][64];
  const int R = a.rows, lane = threadIdx.x & 63, id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = id % WAVES;
  const long long row = (long long)blockIdx.x * (4 / WAVES) + id / WAVES;
  if (row >= (long long)a.batch * a.kv_heads * R) return;      // (WAVES = 1 only, where no barrier follows)
  const int base = (int)(row / R), r = (int)(row - (long long)base * R), b = base / a.kv_heads, hk = base - b * a.kv_heads;
  int gi;
  const int query = query_of(a, r, gi), head = hk * a.group + gi;
  const long long step = 2 * (long long)R * (a.dv + 2);
  const float* from[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) from[m] = a.work + base * a.splits * step + (m * (long long)R + r) * (a.dv + 2);
  f32x2 x[2][BATCH];
  auto load = [&](int c0, int s0) {      // (a row of the workspace is dv + 2 floats: the second of a pair is there for the last column too)
    const int col = min(c0 + 2 * lane, a.dv - 1);
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (s0 + WAVES * u < a.splits) {
#pragma unroll
        for (int m = 0; m < 2; ++m) __builtin_memcpy(&x[m][u], from[m] + (s0 + WAVES * u) * step + col, 8);
      }
  };
  load(0, wave);
  float weight[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    float top = -INFINITY, sum = 0.0f;
    if (lane < a.splits) {
      top = from[m][lane * step + a.dv];
      sum = from[m][lane * step + a.dv + 1];
    }
    const float high = wave_max(top), ref = high == -INFINITY ? 0.0f : high;
    weight[m] = __builtin_amdgcn_exp2f(top - ref);
    const float total = wave_sum(sum * weight[m]);
    weight[m] *= total != 0.0f ? 1.0f / total : 0.0f;
    if (a.lse != nullptr && wave == 0 && lane == 0) a.lse[(base * 2LL + m) * R + r] = total != 0.0f ? high + __log2f(total) : INFINITY;
  }
  const float lam = lam_at<T>(a, head);
  T* out = reinterpret_cast<T*>(a.o) + o_at(a, b, query, head);
  float* maps = a.maps + o_at(a, b, query, head);
  for (int c0 = 0; c0 < a.dv; c0 += 128) {      // (uniform over a row's waves)
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};      // two columns of map 0, two of map 1
    for (int s0 = wave; s0 < a.splits; s0 += WAVES * BATCH) {
      if (c0 > 0 || s0 >= WAVES * BATCH) load(c0, s0);
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (s0 + WAVES * u < a.splits) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float f = __shfl(weight[m], s0 + WAVES * u);
            acc[2 * m] += x[m][u][0] * f;
            acc[2 * m + 1] += x[m][u][1] * f;
          }
        }
    }
    if constexpr (WAVES > 1) {
      if (c0 > 0) __syncthreads();
      part[wave][lane] = acc;
      __syncthreads();
    }
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < WAVES; ++w) acc += part[w][lane];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = c0 + 2 * lane + e;
        if (col < a.dv) {
          out[col] = (T)(acc[e] - lam * acc[2 + e]);
          if (a.maps != nullptr) {
            maps[col] = acc[e];
            maps[maps_plane(a) + col] = acc[2 + e];
          }
        }
      }
    }
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------
// D_1 = dO . O_1 and D_2 = dO . O_2 of every row (16 lanes per row), of the maps' own unrounded products; bound by bytes: 25 us for 134 MB
// of products and 34 of dO (6.7 TB/s, partly cached)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void rowdot_kernel(const Args a) {
  constexpr int N = Vec<T>::N;
  const int R = a.rows, lane = threadIdx.x & 15;
  const long long all = (long long)a.batch * a.kv_heads * R;
  for (long long w = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); w < all; w += gridDim.x * 16LL) {
    const long long base = w / R;
    const int r = (int)(w - base * R), b = (int)base / a.kv_heads, hk = (int)base - b * a.kv_heads;
    int gi;
    const int query = query_of(a, r, gi), head = hk * a.group + gi;
    const long long at = o_at(a, b, query, head);
    const char* go = reinterpret_cast<const char*>(a.d_o) + at * sizeof(T);
    const char* maps[2] = {reinterpret_cast<const char*>(a.maps + at), reinterpret_cast<const char*>(a.maps + maps_plane(a) + at)};
    float s[2] = {0.0f, 0.0f};
    for (int c = lane; c * N < a.dv; c += 16) {
      float x[N], y[4];
      Vec<T>::unpack(load_chunk<T, VEC>(go, c, a.dv), x);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int u = 0; u < N / 4; ++u) {
          Vec<float>::unpack(load_chunk<float, VEC>(maps[m], c * (N / 4) + u, a.dv), y);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m] += x[4 * u + e] * y[e];
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      s[m] = sum_over_r16(s[m]);
      if (lane == 0) a.dots[(base * 2 + m) * R + r] = s[m];
    }
  }
}

// dlam_h = - sum over samples and queries of sum_j P_2 dP (dq_kernel's unrounded sums; one workgroup per head, fixed order).
// One chain of loads and a tree: 5 - 7 us, latency.
template <typename T>
__global__ __launch_bounds__(1024) void dlam_kernel(const Args a) {
  __shared__ float part[16];
  const int h = blockIdx.x, hk = h / a.group, gi = h % a.group, R = a.rows;
  float s = 0.0f;
  const unsigned total = (unsigned)a.batch * (unsigned)a.nq;      // (below 2^31, as the rows of all heads are)
  for (unsigned x0 = threadIdx.x; x0 < total; x0 += 4096) {
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned x = x0 + u * 1024, b = x / (unsigned)a.nq, i = x - b * (unsigned)a.nq;
      v[u] = x < total ? a.dots[(2LL * a.batch * a.kv_heads + b * a.kv_heads + hk) * R + i * a.group + gi] : 0.0f;
    }
    s += (v[0] + v[1]) + (v[2] + v[3]);
  }
  s = sum_over_r(s);
  s += other_half(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.0f;
    for (int w = 0; w < 16; ++w) t += part[w];
    if (a.lam_type == TYPE_F32) reinterpret_cast<float*>(a.dlam)[h] = -t;
    else reinterpret_cast<T*>(a.dlam)[h] = (T)-t;
  }
}

// dK, dV of 32 keys per wave: grid (key tiles x row splits x kv_heads x batch), GROUPS x 2 waves.  row_splits > 1: the rows that see a key tile
// are cut into equal parts, whose sums meet in the workspace (key_join_kernel): with a causal mask the first keys are seen by all rows and
// the last by few, and one workgroup per key tile would leave half the chip idle half the time.
// Both waves run the same code on (lse, D): map 1's weight is taken as +|lam| P_2 with |lam| folded into lse, and its results are negated when they
// leave the wave.  Only where a lam of the group is negative do its rows' signs have to be put back (flip).
// Bound by matrix instructions: (2, 4096, 16 / 4 heads, 64 / 128, bf16, "start") 700 us = 0.88 PFLOP/s executed (lam applied to each weight cost 47 more);
// (5, 517 x 1531, 6 / 2, 128 / 256, fp16) 174 us, 480 workgroups of 64 keys and half of the rows, of which 8 in 10 have keys; (128, 190, 1, 32 / 64, fp32) 49 us.
template <typename T, int D, bool VEC>
__global__ __launch_bounds__((128 * key_groups<T, D>())) __attribute__((amdgpu_waves_per_eu(D * sizeof(T) <= 128 ? 2 : 1))) void dkv_kernel(const Args a) {
  constexpr int GROUPS = key_groups<T, D>(), NTH = 128 * GROUPS, KEYS = 32 * GROUPS;
  constexpr int DV = 2 * D, RT = 32, NT = D / 32, NTV = DV / 32, NJ = D / (2 * Vec<T>::N), SZ = sizeof(T);
  constexpr int QB = Tile<T, D>::bytes(RT), OB = Tile<T, DV>::bytes(RT), BUF = 2 * QB + OB;
  __shared__ __align__(16) char lds[2 * BUF], vt[Tile<T, DV>::bytes(KEYS)];      // row tiles; the workgroup's own values
  __shared__ __align__(16) float stat[2][2][3][RT];      // [buffer][map][lse - log2 |coefficient|, D, its sign] of the tile's rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ki = lane & 31, g = lane >> 5;
  const int group = wave >> 1, map = wave & 1;
  const int R = a.rows, tiles = (a.nk + KEYS - 1) / KEYS;
  int base, unit;
  grid_order(blockIdx.x, a.batch * a.kv_heads, tiles * a.row_splits, base, unit);
  const int split = unit % a.row_splits, tile = unit / a.row_splits;      // the keys that most rows see first
  const int b = base / a.kv_heads, hk = base - b * a.kv_heads;
  const int len = length_of(a, b);
  const int wg_key = tile * KEYS, key0 = wg_key + group * 32, key = key0 + ki;
  const float c = a.scale * 1.44269504088896340736f;
  u32x4_t k[NJ];
  const int q_at = map * QB + Tile<T, D>::rows_at(lane), g_at = 2 * QB + Tile<T, DV>::rows_at(lane);
  const int qt_at = map * QB + Tile<T, D>::columns_at(lane), gt_at = 2 * QB + Tile<T, DV>::columns_at(lane);
  const char* own = vt + Tile<T, DV>::bytes(32) * group + Tile<T, DV>::rows_at(lane);
  f32x16 dk[NT], dv[NTV];
  zero_acc(dk);
  zero_acc(dv);
  ColumnScale<T> range;
  float lift = 0.0f;      // fp16: the weights are taken 2^lift times as large, up to 2^12 (over thousands of keys they lie below its normal range; as in the forward)
  bool flip = false;
  const int seen_from = wg_key < len ? first_query(a, wg_key, len) * a.group / RT * RT : R;
  const int per = ((R - seen_from + a.row_splits - 1) / a.row_splits + RT - 1) / RT * RT;
  const int r_first = seen_from + split * per, r_last = min(R, r_first + per);
  const int wave_first = key0 < len ? first_query(a, key0, len) * a.group : R;
  const int wave_all = key0 + 31 < len ? first_query(a, key0 + 31, len) * a.group : R;      // rows from here on see all 32 keys
  const int my_first = key < len ? first_query(a, key, len) * a.group : R;                   // rows from here on see this lane's key
  if (r_first < r_last) {
    const char* kp = reinterpret_cast<const char*>(a.k) + (b * a.k_b + min(key, len - 1) * a.k_n + (2 * hk + map) * a.k_h) * SZ;
#pragma unroll
    for (int j = 0; j < NJ; ++j) k[j] = load_chunk<T, VEC>(kp, 2 * j + g, a.d);
    {
      typedef Stage<T, DV, KEYS, NTH, VEC> StageV;
      StageV sv;
      unsigned vo[StageV::PER];
      key_offsets<StageV, 1>(vo, tid, (unsigned)a.v_n * SZ, 0, len - 1 - wg_key);
      sv.load(tid, reinterpret_cast<const char*>(a.v) + (b * a.v_b + wg_key * a.v_n + hk * a.v_h) * SZ, vo, a.dv);
      sv.store(tid, vt, a.dv);
    }
    typedef Stage<T, D, 2 * RT, NTH, VEC> StageQ;
    typedef Stage<T, DV, RT, NTH, VEC> StageO;
    StageQ sq;
    StageO so;
    float st = 0.0f;
    const char* qp = reinterpret_cast<const char*>(a.q) + (b * a.q_b + 2 * hk * a.group * a.q_h) * SZ;
    const char* op = reinterpret_cast<const char*>(a.d_o) + o_at(a, b, 0, hk * a.group) * SZ;
    float largest = 1.0f;
    for (int gi = 0; gi < a.group; ++gi) {
      const float lam = lam_at<T>(a, hk * a.group + gi);
      flip = flip || lam < 0.0f;
      largest = fmaxf(largest, fabsf(lam));
    }
    if constexpr (ColumnScale<T>::USED) lift = largest < 0x1p100f ? (float)(12 - __builtin_amdgcn_frexp_expf(largest)) : 0.0f;
    static_assert(NTH >= 6 * RT, "a thread stages one statistic");
    const int sw = tid >> 5, sm = sw >= 3 ? 1 : 0, sk = sw - 3 * sm;      // which statistic of which map
    // a tile of 32 rows holds whole queries where the group divides 32: its rows' offsets then are the same in every tile
    const bool whole = RT % a.group == 0;
    unsigned qo[StageQ::PER], oo[StageO::PER];
    float extra = 0.0f;      // what this thread's statistic takes of lam: -log2 |coefficient| or its sign
    auto offsets = [&](int r0, int i0) {
      row_offsets<StageQ, 2>(a, qo, tid, r0, i0, (unsigned)a.q_n * SZ, 2u * (unsigned)a.q_h * SZ, (unsigned)a.q_h * SZ);
      row_offsets<StageO, 1>(a, oo, tid, r0, i0, (unsigned)(a.heads * a.dv) * SZ, (unsigned)a.dv * SZ, 0);
      int gi;
      query_of(a, min(r0 + (tid & 31), R - 1), gi);
      const float lam = sm == 0 ? 1.0f : lam_at<T>(a, hk * a.group + gi);
      extra = sk == 0 ? -__log2f(fabsf(lam)) - lift : sk == 1 ? 0.0f : lam < 0.0f ? -1.0f : 1.0f;
    };
    offsets(r_first, r_first / a.group);
    auto fetch = [&](int r0) {
      const int i0 = r0 / a.group;
      if (!whole || r0 + RT > R) offsets(r0, i0);
      sq.load(tid, qp + i0 * a.q_n * SZ, qo, a.d);
      so.load(tid, op + (long long)i0 * a.heads * a.dv * SZ, oo, a.dv);
      if (tid < 6 * RT) {
        const int rw = min(r0 + (tid & 31), R - 1);
        if (sk < 2) st = (sk == 0 ? a.lse : a.dots)[((long long)base * 2 + sm) * R + rw];
      }
    };
    auto place = [&](int buf) {
      sq.store(tid, lds + buf * BUF, a.d);
      so.store(tid, lds + buf * BUF + 2 * QB, a.dv);
      if (tid < 6 * RT) (&stat[buf][0][0][0])[tid] = st + extra;
    };
    fetch(r_first);
    place(0);
    __syncthreads();
    two_buffers<RT>(r_first, r_last, [&](int r0, auto which) {
      constexpr int CUR = decltype(which)::value;
      const char* buf = lds + CUR * BUF;
      const bool more = r0 + RT < r_last;
      if (more) fetch(r0 + RT);
      if (r0 + RT > wave_first) {
        f32x16 w = mm_tile<T, D>(buf + q_at, k), ds = mm_tiles<T, DV>(buf + g_at, own);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 l = *reinterpret_cast<const f32x4*>(&stat[CUR][map][0][8 * u + 4 * g]);
          const f32x4 dd = *reinterpret_cast<const f32x4*>(&stat[CUR][map][1][8 * u + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = 4 * u + e;
            w[t] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[t], c, -l[e]));
            ds[t] = w[t] * (ds[t] - dd[e]);
          }
        }
        if (flip) {
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const float f = stat[CUR][map][2][tile_row(t, g)];
            w[t] *= f;
            ds[t] *= f;
          }
        }
        if (r0 < wave_all || r0 + RT > R) {      // (the products are replaced, not the factors: nothing that stands in a hidden place gets through)
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const int row = r0 + tile_row(t, g);
            const bool seen = row >= my_first && row < R;
            w[t] = seen ? w[t] : 0.0f;
            ds[t] = seen ? ds[t] : 0.0f;
          }
        }
        mm_transposed<T, DV, NTV>(dv, buf + gt_at, w);
        range.fit(ds, dk);
        mm_transposed<T, D, NT>(dk, buf + qt_at, ds);
      }
      if (more) {
        place(CUR ^ 1);
        __syncthreads();
      }
    });
  }
  const bool live = key < len, there = key < a.nk;      // (rows behind the length: the clamped key's sums are not theirs)
  const long long at = ((long long)b * a.nk + key) * a.kv_heads + hk;
  const int width = 2 * a.d + a.dv;
  const float lower = __builtin_amdgcn_exp2f(-lift), back = lower / range.factor;
  float* part = a.work + ((long long)split * a.batch * a.nk * a.kv_heads + at) * width;      // [split][sample, key, head][dk1 | dk2 | dv]
  auto put = [&](int which, int col, f32x4 x) {
    if (!there) return;
    if (!live) x = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.row_splits > 1) store4<float, VEC>(part + which * a.d, col, which < 2 ? a.d : a.dv, x);
    else store4<T, VEC>(which < 2 ? reinterpret_cast<T*>(a.dk) + (at * 2 + which) * a.d : reinterpret_cast<T*>(a.dv_out) + at * a.dv, col, which < 2 ? a.d : a.dv, x);
  };
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dk[t][4 * u + e] * back * (map == 0 ? a.scale : -a.scale);
      put(map, 32 * t + 8 * u + 4 * g, x);
    }
  hand_over<NTV, GROUPS, 2 * BUF>(dv, lds, group, map, lane, [&](int t, const f32x16& x, const f32x16& y) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 z;
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = (x[4 * u + e] - y[4 * u + e]) * lower;
      put(2, 32 * t + 8 * u + 4 * g, z);
    }
  });
}

// dK, dV = the row splits' sums, in order; a thread per four elements (VEC) or one; bytes: 13.7 us for 50 MB in, 8 out
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void key_join_kernel(const Args a) {
  constexpr int N = VEC ? 4 : 1;
  const int w = 2 * a.d + a.dv, items = w / N;
  const long long all = (long long)a.batch * a.nk * a.kv_heads, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= all * items) return;
  const long long at = i / items;
  const int col = (int)(i - at * items) * N;
  float x[N];
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = 0.0f;
  for (int s = 0; s < a.row_splits; ++s) {
    const float* part = a.work + (s * all + at) * w + col;
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] += part[e];
  }
  T* out = col < 2 * a.d ? reinterpret_cast<T*>(a.dk) + at * 2 * a.d + col : reinterpret_cast<T*>(a.dv_out) + at * a.dv + (col - 2 * a.d);
  if constexpr (VEC) store4<T, true>(out, 0, 4, f32x4{x[0], x[1], x[2], x[3]});
  else *out = (T)x[0];
}

// dQ of 32 rows per wave: grid (row tiles x kv_heads x batch), GROUPS x 2 waves; dO of the workgroup's rows stays in LDS (the registers hold
// Q, the sums and two tiles of scores).  Bound by matrix instructions: (2, 4096, 16 / 4 heads, 64 / 128, bf16, "start") 433 us = 0.79 PFLOP/s executed;
// (5, 517 x 1531, 6 / 2, 128 / 256, fp16) 108 us; (128, 190, 1, 32 / 64, fp32) 32 us.
template <typename T, int D, bool VEC>
__global__ __launch_bounds__((128 * dq_groups<T, D>())) __attribute__((amdgpu_waves_per_eu(2))) void dq_kernel(const Args a) {
  constexpr int GROUPS = dq_groups<T, D>(), NTH = 128 * GROUPS, ROWS = 32 * GROUPS;
  constexpr int DV = 2 * D, KT = 32, NT = D / 32, NJ = D / (2 * Vec<T>::N), SZ = sizeof(T);
  constexpr int KB = Tile<T, D>::bytes(KT), VB = Tile<T, DV>::bytes(KT), BUF = 2 * KB + VB;
  __shared__ __align__(16) char lds[2 * BUF], gt[Tile<T, DV>::bytes(ROWS)];      // key tiles; dO of the workgroup's own rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 31, g = lane >> 5;
  const int group = wave >> 1, map = wave & 1;
  const int R = a.rows, tiles = (R + ROWS - 1) / ROWS;
  int base, unit;
  grid_order(blockIdx.x, a.batch * a.kv_heads, tiles, base, unit);
  const int tile = tiles - 1 - unit;
  const int b = base / a.kv_heads, hk = base - b * a.kv_heads;
  const int len = length_of(a, b);
  const int row0 = tile * ROWS + group * 32, r = row0 + qi, rr = r < R ? r : R - 1;
  int gi;
  const int query = query_of(a, rr, gi), head = hk * a.group + gi;
  const int wg_end = end_of(a, (min((tile + 1) * ROWS, R) - 1) / a.group, len);
  const int my_end = r < R ? end_of(a, query, len) : 0;
  const int wave_end = row0 < R ? end_of(a, min(row0 + 31, R - 1) / a.group, len) : 0;
  const int wave_all = row0 + 31 < R ? end_of(a, row0 / a.group, len) : 0;
  const float c = a.scale * 1.44269504088896340736f;
  u32x4_t q[NJ];
  const char* qp = reinterpret_cast<const char*>(a.q) + (b * a.q_b + query * a.q_n + (2 * head + map) * a.q_h) * SZ;
#pragma unroll
  for (int j = 0; j < NJ; ++j) q[j] = load_chunk<T, VEC>(qp, 2 * j + g, a.d);
  {
    typedef Stage<T, DV, ROWS, NTH, VEC> StageG;
    StageG sg;
    unsigned offset[StageG::PER];
    const int r0 = tile * ROWS, i0 = r0 / a.group;
    row_offsets<StageG, 1>(a, offset, tid, r0, i0, (unsigned)(a.heads * a.dv) * SZ, (unsigned)a.dv * SZ, 0);
    sg.load(tid, reinterpret_cast<const char*>(a.d_o) + o_at(a, b, i0, hk * a.group) * SZ, offset, a.dv);
    sg.store(tid, gt, a.dv);      // (read behind the barrier that follows the first key tile)
  }
  const long long at = ((long long)base * 2 + map) * R + rr;
  const float l = a.lse[at], dd = a.dots[at], cf = map == 0 ? 1.0f : -lam_at<T>(a, head);
  float dot = 0.0f;      // sum_j P dP: map 1's is what dlam is made of
  const int k_at = map * KB + Tile<T, D>::rows_at(lane), kt_at = map * KB + Tile<T, D>::columns_at(lane), v_at = 2 * KB + Tile<T, DV>::rows_at(lane);
  const char* own = gt + Tile<T, DV>::bytes(32) * group + Tile<T, DV>::rows_at(lane);
  f32x16 dq[NT];
  zero_acc(dq);
  ColumnScale<T> range;
  typedef Stage<T, D, 2 * KT, NTH, VEC> StageK;
  typedef Stage<T, DV, KT, NTH, VEC> StageV;
  StageK sk;
  StageV sv;
  const char* kp = reinterpret_cast<const char*>(a.k) + (b * a.k_b + 2 * hk * a.k_h) * SZ;
  const char* vp = reinterpret_cast<const char*>(a.v) + (b * a.v_b + hk * a.v_h) * SZ;
  auto fetch = [&](int j0) {
    unsigned ko[StageK::PER], vo[StageV::PER];
    key_offsets<StageK, 2>(ko, tid, (unsigned)a.k_n * SZ, (unsigned)a.k_h * SZ, wg_end - 1 - j0);
    key_offsets<StageV, 1>(vo, tid, (unsigned)a.v_n * SZ, 0, wg_end - 1 - j0);
    sk.load(tid, kp + j0 * a.k_n * SZ, ko, a.d);
    sv.load(tid, vp + j0 * a.v_n * SZ, vo, a.dv);
  };
  auto place = [&](char* buf) {
    sk.store(tid, buf, a.d);
    sv.store(tid, buf + 2 * KB, a.dv);
  };
  if (wg_end > 0) {
    fetch(0);
    place(lds);
    __syncthreads();
    two_buffers<KT>(0, wg_end, [&](int j0, auto which) {
      constexpr int CUR = decltype(which)::value;
      const char* buf = lds + CUR * BUF;
      const bool more = j0 + KT < wg_end;
      if (more) fetch(j0 + KT);
      if (j0 < wave_end) {
        f32x16 w = mm_tile<T, D>(buf + k_at, q), ds = mm_tiles<T, DV>(buf + v_at, own);
#pragma unroll
        for (int t = 0; t < 16; ++t) w[t] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[t], c, -l));
        if (j0 + KT > wave_all) {
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const bool seen = j0 + tile_row(t, g) < my_end;
            w[t] = seen ? w[t] : 0.0f;
            ds[t] = seen ? ds[t] : 0.0f;
          }
        }
        if (map == 1) {
          float s = 0.0f;
#pragma unroll
          for (int t = 0; t < 16; ++t) s = __builtin_fmaf(w[t], ds[t], s);
          dot += s;
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) ds[t] = w[t] * (ds[t] - dd);
        if (j0 + KT > wave_all) {      // (dd may be no number where the row sees nothing)
#pragma unroll
          for (int t = 0; t < 16; ++t) ds[t] = j0 + tile_row(t, g) < my_end ? ds[t] : 0.0f;
        }
        range.fit(ds, dq);
        mm_transposed<T, D, NT>(dq, buf + kt_at, ds);
      }
      if (more) {
        place(lds + (CUR ^ 1) * BUF);
        __syncthreads();
      }
    });
  }
  dot += other_half(dot);
  if (r >= R) return;
  if (map == 1 && g == 0) a.dots[(2LL * a.batch * a.kv_heads + base) * R + r] = dot;
  T* out = reinterpret_cast<T*>(a.dq) + ((((long long)b * a.nq + query) * a.heads + head) * 2 + map) * a.d;
  const float f = a.scale * cf, back = 1.0f / range.factor;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dq[t][4 * u + e] * back * f;
      store4<T, VEC>(out, 32 * t + 8 * u + 4 * g, a.d, x);
    }
}

// ---- launches: one compilation unit per element type ----------------------------------------------------------------------------------
template <typename T, int D, bool VEC>
void launch_fwd(const Args& a, hipStream_t st) {
  const int heads = a.kv_heads * a.batch;
  if (a.rows <= 32) {      // a handful of rows: one pair of waves per workgroup, the keys split over many of them
    fwd_kernel<T, D, 1, VEC><<<a.splits * heads, 128, 0, st>>>(a);
  } else {
    constexpr int GROUPS = fwd_groups<T, D>(), ROWS = 32 * GROUPS;
    fwd_kernel<T, D, GROUPS, VEC><<<(a.rows + ROWS - 1) / ROWS * a.splits * heads, 4 * ROWS, 0, st>>>(a);
  }
  if (a.splits > 1) {
    if (a.rows <= 32) join_kernel<T, 4><<<heads * a.rows, 256, 0, st>>>(a);
    else join_kernel<T, 1><<<(unsigned)(((long long)heads * a.rows + 3) / 4), 256, 0, st>>>(a);
  }
}

template <typename T, int D, bool VEC>
void launch_bwd(const Args& a, hipStream_t st) {
  const int heads = a.kv_heads * a.batch;
  constexpr int KEYS = 32 * key_groups<T, D>(), ROWS = 32 * dq_groups<T, D>();
  const long long sums = ((long long)heads * a.rows + 15) / 16;
  rowdot_kernel<T, VEC><<<(unsigned)(sums < 1 << 23 ? sums : 1 << 23), 256, 0, st>>>(a);      // (a launch of 2^24 workgroups runs short of them)
  if (a.dk != nullptr) dkv_kernel<T, D, VEC><<<(a.nk + KEYS - 1) / KEYS * a.row_splits * heads, 4 * KEYS, 0, st>>>(a);
  if (a.dk != nullptr && a.row_splits > 1)
    key_join_kernel<T, VEC><<<(unsigned)(((long long)heads * a.nk * (2 * a.d + a.dv) / (VEC ? 4 : 1) + 255) / 256), 256, 0, st>>>(a);
  if (a.dq != nullptr) dq_kernel<T, D, VEC><<<(a.rows + ROWS - 1) / ROWS * heads, 4 * ROWS, 0, st>>>(a);
  if (a.dlam != nullptr) dlam_kernel<T><<<a.heads, 1024, 0, st>>>(a);
}

// the built width a call runs at: heads of at most D elements, values of at most 2 D (shorter rows are padded with zeros on chip);
// 0: wider than any.  32-bit inputs stop at 64 / 128: the resident operands of wider heads do not fit a wave's 512 registers.
// Rows that cannot be read in 16-byte chunks (odd sizes, strides or pointers) run element by element at the widest.
inline int class_of(const Args& a) {
  const int need = a.d > (a.dv + 1) / 2 ? a.d : (a.dv + 1) / 2, most = a.type == TYPE_F32 ? 64 : 128;
  return need > most ? 0 : !a.vec ? most : need <= 32 ? 32 : need <= 64 ? 64 : 128;
}

template <typename T, int D, bool VEC>
void launch(const Args& a, bool backward, hipStream_t st) {
  if (backward) launch_bwd<T, D, VEC>(a, st);
  else launch_fwd<T, D, VEC>(a, st);
}

void run_f32(const Args& a, bool backward, hipStream_t st);
void run_bf16(const Args& a, bool backward, hipStream_t st);
void run_f16(const Args& a, bool backward, hipStream_t st);

}  // namespace da
}  // namespace is
