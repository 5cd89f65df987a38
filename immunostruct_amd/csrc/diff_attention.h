// Differential attention: o_i = sum_j (P1 - lam P2)_ij v_j, P_m = softmax_j(scale q_m,i . k_m,j) over the keys that query i sees.
//
//   rows      the queries of one (sample, key head) and its G = heads / kv_heads query heads are packed into R = nq G rows, row r = query
//             r / G, head r % G of the group: a key tile is read once for all heads that share it, and the gradients of shared keys
//             are sums inside one workgroup (no atomics anywhere; every result has one fixed summation order).
//   visible   key j < end(i): end = len (no mask), min(len, i + 1) ("start") or len - nq + 1 + i ("end").  Keys at or behind len are never
//             read (their rows are clamped to the last valid one and their scores replaced), so anything may stand there.
//             A row that sees nothing gives 0, lse = +inf, and no gradient.
//   forward   one pass over the keys: S^T = K Q^T (a lane owns one query), running maximum and sum per map in 32 bits, O^T += V^T P^T for
//             both maps from ONE transposed read of V.  The maximum only moves when a score passes it by 2^8 (the weights stay <= 2^8, far
//             inside every type), which makes the rescaling of the two accumulators rare.
//   backward  dP = dO V^T is shared by the maps; D_m = dO . O_m; dS_1 = P1 (dP - D_1), dS_2 = -lam P2 (dP - D_2);
//             dQ_m = scale dS_m K_m, dK_m = scale dS_m^T Q_m, dV = (P1 - lam P2)^T dO, dlam = -sum D_2.  Scores are recomputed from lse.
//             dK / dV: a wave owns 32 keys and walks the rows; dQ: a wave owns 32 rows and walks the keys.
// Scores, sums, lse, D and all accumulators are 32-bit; P and dS are rounded once to the inputs' type for the matrix instructions.
#pragma once
#include "../../include/immunostruct_hip.h"
#include "tiles16.h"

namespace is {
namespace da {

typedef IsDiffAttention Args;
constexpr float SLACK = 8.0f;      // log2 of how far a weight may pass 1 before the running maximum follows

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

// byte offsets of a tile's key rows j0 + row_of(k), clamped to the last valid one, from row j0
template <typename S>
__device__ __forceinline__ void key_offsets(unsigned (&out)[S::PER], int tid, unsigned stride, int left) {
#pragma unroll
  for (int k = 0; k < S::PER; ++k) out[k] = (unsigned)min(S::row_of(tid, k), left) * stride;
}
// byte offsets of a tile's packed rows r0 + row_of(k), clamped to the last one, from query r0 / group and the group's first head
template <typename S>
__device__ __forceinline__ void row_offsets(const Args& a, unsigned (&out)[S::PER], int tid, int r0, int first, unsigned stride, unsigned head) {
#pragma unroll
  for (int k = 0; k < S::PER; ++k) {
    int g;
    const int i = query_of(a, min(r0 + S::row_of(tid, k), a.rows - 1), g);
    out[k] = (unsigned)(i - first) * stride + (unsigned)g * head;
  }
}

// ---- forward -----------------------------------------------------------------------------------------------------------------------
// grid: (row tiles x splits x kv_heads x batch), NW waves of 32 rows.  splits > 1: every workgroup takes one range of the keys and leaves
// unnormalised sums with their maxima in the workspace; join_kernel puts them together.
template <typename T, int D, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW, (D <= 64 && NW > 1 ? 2 : 1)) void fwd_kernel(const Args a) {
  constexpr int DV = 2 * D, KT = 32, NT = DV / 32, NJ = D / (2 * Vec<T>::N), NTH = 64 * NW, SZ = sizeof(T);
  constexpr int KB = Tile<T, D>::bytes(KT), VB = Tile<T, DV>::bytes(KT), BUF = 2 * KB + VB;
  __shared__ __align__(16) char lds[2 * BUF];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 31, g = lane >> 5;
  const int R = a.rows, tiles = (R + 32 * NW - 1) / (32 * NW);
  int base, unit;
  grid_order(blockIdx.x, a.batch * a.kv_heads, tiles * a.splits, base, unit);
  const int split = unit % a.splits, tile = tiles - 1 - unit / a.splits;      // the rows that see most keys first
  const int b = base / a.kv_heads, hk = base - b * a.kv_heads;
  const int len = length_of(a, b);
  const int row0 = tile * 32 * NW + wave * 32, r = row0 + qi, rr = r < R ? r : R - 1;
  int gi;
  const int query = query_of(a, rr, gi), head = hk * a.group + gi;
  const int wg_end = end_of(a, (min(tile * 32 * NW + 32 * NW, R) - 1) / a.group, len);
  const int my_end = r < R ? end_of(a, query, len) : 0;
  const int wave_end = row0 < R ? end_of(a, min(row0 + 31, R - 1) / a.group, len) : 0;      // no row of the wave sees further
  const int wave_all = row0 + 31 < R ? end_of(a, row0 / a.group, len) : 0;                  // every row of the wave sees this far
  const int per = ((wg_end + a.splits - 1) / a.splits + KT - 1) / KT * KT;
  const int first = split * per, last = min(wg_end, first + per);
  const float c = a.scale * 1.44269504088896340736f;

  u32x4_t q[2][NJ];
  const char* qp = reinterpret_cast<const char*>(a.q) + (b * a.q_b + query * a.q_n + 2 * head * a.q_h) * SZ;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j) q[m][j] = load_chunk<T, VEC>(qp + m * a.q_h * SZ, 2 * j + g, a.d);
  f32x16 o[2][NT];
  zero_acc2(o);
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

  typedef Stage<T, D, KT, NTH, VEC> StageK;
  typedef Stage<T, DV, KT, NTH, VEC> StageV;
  StageK sk0, sk1;
  StageV sv;
  const char* kp = reinterpret_cast<const char*>(a.k) + (b * a.k_b + 2 * hk * a.k_h) * SZ;
  const char* vp = reinterpret_cast<const char*>(a.v) + (b * a.v_b + hk * a.v_h) * SZ;
  auto fetch = [&](int j0) {
    unsigned ko[StageK::PER], vo[StageV::PER];
    key_offsets<StageK>(ko, tid, (unsigned)a.k_n * SZ, len - 1 - j0);
    key_offsets<StageV>(vo, tid, (unsigned)a.v_n * SZ, len - 1 - j0);
    const char* k = kp + j0 * a.k_n * SZ;
    sk0.load(tid, k, ko, a.d);
    sk1.load(tid, k + a.k_h * SZ, ko, a.d);
    sv.load(tid, vp + j0 * a.v_n * SZ, vo, a.dv);
  };
  auto place = [&](char* buf) {
    sk0.store(tid, buf);
    sk1.store(tid, buf + KB);
    sv.store(tid, buf + 2 * KB);
  };
  if (first < last) {      // (uniform over the workgroup, as is every barrier below)
    fetch(first);
    place(lds);
    __syncthreads();
    int cur = 0;
    for (int j0 = first; j0 < last; j0 += KT) {
      const bool more = j0 + KT < last;
      if (more) fetch(j0 + KT);
      if (j0 < wave_end) {
        const char* buf = lds + cur * BUF;
        f32x16 p[2];
        zero_acc(p);
        mm_tile<T, D>(p[0], buf, 0, q[0], lane);
        mm_tile<T, D>(p[1], buf + KB, 0, q[1], lane);
        if (j0 + KT > wave_all) {
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const bool hidden = j0 + tile_row(t, g) >= my_end;
            p[0][t] = hidden ? -INFINITY : p[0][t];
            p[1][t] = hidden ? -INFINITY : p[1][t];
          }
        }
        float high[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float x = p[m][0];
#pragma unroll
          for (int t = 1; t < 16; ++t) x = fmaxf(x, p[m][t]);
          high[m] = fmaxf(x, other_half(x));
        }
        if (__any((high[0] - top[0]) * c > SLACK || (high[1] - top[1]) * c > SLACK)) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float now = fmaxf(top[m], high[m]), ref = now == -INFINITY ? 0.0f : now;
            const float shrink = __builtin_amdgcn_exp2f((top[m] - ref) * c);
            top[m] = now;
            sum[m] *= shrink;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 16; ++e) o[m][t][e] *= shrink;
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float ref = top[m] == -INFINITY ? 0.0f : -top[m] * c;
          float s = 0.0f;
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            p[m][t] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[m][t], c, ref));
            s += p[m][t];
          }
          sum[m] += s;
        }
        mm_transposed<T, DV, NT, 2>(o, buf + 2 * KB, 0, p, lane);
      }
      if (more) {
        place(lds + (cur ^ 1) * BUF);
        __syncthreads();
        cur ^= 1;
      }
    }
  }
  float total[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) total[m] = sum[m] + other_half(sum[m]);
  if (r >= R) return;
  if (a.splits > 1) {
    float* w = a.work + ((long long)base * a.splits + split) * (2 * (long long)R * (a.dv + 2));
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float* wm = w + (m * (long long)R + r) * (a.dv + 2);
      if (g == 0) {
        wm[a.dv] = top[m] == -INFINITY ? -INFINITY : top[m] * c;
        wm[a.dv + 1] = total[m];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          store4<float, false>(wm, 32 * t + 8 * u + 4 * g, a.dv, f32x4{o[m][t][4 * u], o[m][t][4 * u + 1], o[m][t][4 * u + 2], o[m][t][4 * u + 3]});
    }
    return;
  }
  const float lam = lam_at<T>(a, head);
  const float w0 = total[0] != 0.0f ? 1.0f / total[0] : 0.0f, w1 = total[1] != 0.0f ? 1.0f / total[1] : 0.0f;
  if (a.lse != nullptr && g == 0) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
      a.lse[((long long)base * 2 + m) * R + r] = total[m] != 0.0f ? __builtin_fmaf(top[m], c, __log2f(total[m])) : INFINITY;
  }
  T* out = reinterpret_cast<T*>(a.o) + o_at(a, b, query, head);
  T* out2 = reinterpret_cast<T*>(a.o2) + o_at(a, b, query, head);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = o[1][t][4 * u + e] * w1;
        x[e] = o[0][t][4 * u + e] * w0 - lam * y[e];
      }
      store4<T, VEC>(out, 32 * t + 8 * u + 4 * g, a.dv, x);
      if (a.o2 != nullptr) store4<T, VEC>(out2, 32 * t + 8 * u + 4 * g, a.dv, y);
    }
}

// the splits of one row put together: one wave per row, lane = column
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  const int R = a.rows, lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (long long)a.batch * a.kv_heads * R) return;
  const long long base = w / R;
  const int r = (int)(w - base * R), b = (int)base / a.kv_heads, hk = (int)base - b * a.kv_heads;
  int gi;
  const int query = query_of(a, r, gi), head = hk * a.group + gi;
  float inv[2], top[2], total[2];
  const long long step = 2 * (long long)R * (a.dv + 2);
  const float* from[2];
  for (int m = 0; m < 2; ++m) {
    from[m] = a.work + base * a.splits * step + (m * (long long)R + r) * (a.dv + 2);
    top[m] = -INFINITY;
    total[m] = 0.0f;
    for (int s = 0; s < a.splits; ++s) top[m] = fmaxf(top[m], from[m][s * step + a.dv]);
    const float ref = top[m] == -INFINITY ? 0.0f : top[m];
    for (int s = 0; s < a.splits; ++s) total[m] += from[m][s * step + a.dv + 1] * __builtin_amdgcn_exp2f(from[m][s * step + a.dv] - ref);
    inv[m] = total[m] != 0.0f ? 1.0f / total[m] : 0.0f;
    if (a.lse != nullptr && lane == 0) a.lse[(base * 2 + m) * R + r] = total[m] != 0.0f ? top[m] + __log2f(total[m]) : INFINITY;
  }
  const float lam = lam_at<T>(a, head);
  T* out = reinterpret_cast<T*>(a.o) + o_at(a, b, query, head);
  T* out2 = reinterpret_cast<T*>(a.o2) + o_at(a, b, query, head);
  for (int col = lane; col < a.dv; col += 64) {
    float x[2];
    for (int m = 0; m < 2; ++m) {
      const float ref = top[m] == -INFINITY ? 0.0f : top[m];
      float acc = 0.0f;
      for (int s = 0; s < a.splits; ++s) acc += from[m][s * step + col] * __builtin_amdgcn_exp2f(from[m][s * step + a.dv] - ref);
      x[m] = acc * inv[m];
    }
    out[col] = (T)(x[0] - lam * x[1]);
    if (a.o2 != nullptr) out2[col] = (T)x[1];
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------
// D_2 = dO . O_2 and D_1 = dO . O + lam D_2 of every row (one wave per row)
template <typename T>
__global__ __launch_bounds__(256) void rowdot_kernel(const Args a) {
  const int R = a.rows, lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (long long)a.batch * a.kv_heads * R) return;
  const long long base = w / R;
  const int r = (int)(w - base * R), b = (int)base / a.kv_heads, hk = (int)base - b * a.kv_heads;
  int gi;
  const int query = query_of(a, r, gi), head = hk * a.group + gi;
  const long long at = o_at(a, b, query, head);
  const T *o = reinterpret_cast<const T*>(a.o) + at, *o2 = reinterpret_cast<const T*>(a.o2) + at, *go = reinterpret_cast<const T*>(a.d_o) + at;
  float s = 0.0f, s2 = 0.0f;
  for (int col = lane; col < a.dv; col += 64) {
    const float x = (float)go[col];
    s += x * (float)o[col];
    s2 += x * (float)o2[col];
  }
  s = sum_over_r(s);
  s2 = sum_over_r(s2);
  s += other_half(s);
  s2 += other_half(s2);
  if (lane == 0) {
    a.dots[(base * 2) * R + r] = s + lam_at<T>(a, head) * s2;
    a.dots[(base * 2 + 1) * R + r] = s2;
  }
}

// dlam_h = - sum over samples and queries of sum_j P_2 dP (dq_kernel's unrounded sums; one workgroup per head, fixed order)
template <typename T>
__global__ __launch_bounds__(1024) void dlam_kernel(const Args a) {
  __shared__ float part[16];
  const int h = blockIdx.x, hk = h / a.group, gi = h % a.group, R = a.rows;
  float s = 0.0f;
  for (long long x = threadIdx.x; x < (long long)a.batch * a.nq; x += 1024) {
    const long long b = x / a.nq;
    const int i = (int)(x - b * a.nq);
    s += a.dots[(2LL * a.batch * a.kv_heads + b * a.kv_heads + hk) * R + i * a.group + gi];
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

// dK, dV of 32 keys per wave: grid (key tiles x row splits x kv_heads x batch).  row_splits > 1: the rows that see a key tile are cut into equal
// parts, whose sums meet in the workspace (key_join_kernel): with a causal mask the first keys are seen by all rows and the last by few, and a
// workgroup of 512-register waves is alone on its CU, so one workgroup per key tile would leave half the chip idle half the time.
template <typename T, int D, bool VEC>
__global__ __launch_bounds__(256, 1) void dkv_kernel(const Args a) {
  constexpr int DV = 2 * D, RT = 32, NT = D / 32, NTV = DV / 32, NJ = D / (2 * Vec<T>::N), NJV = DV / (2 * Vec<T>::N), SZ = sizeof(T);
  constexpr int QB = Tile<T, D>::bytes(RT), OB = Tile<T, DV>::bytes(RT), BUF = 2 * QB + OB;
  __shared__ __align__(16) char lds[2 * BUF];
  __shared__ __align__(16) float stat[2][5][RT];      // lse1, lse2, D1, D2, lam of the tile's rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ki = lane & 31, g = lane >> 5;
  const int R = a.rows, tiles = (a.nk + 127) / 128;
  int base, unit;
  grid_order(blockIdx.x, a.batch * a.kv_heads, tiles * a.row_splits, base, unit);
  const int split = unit % a.row_splits, tile = unit / a.row_splits;      // the keys that most rows see first
  const int b = base / a.kv_heads, hk = base - b * a.kv_heads;
  const int len = length_of(a, b);
  const int wg_key = tile * 128, key0 = wg_key + wave * 32, key = key0 + ki;
  const float c = a.scale * 1.44269504088896340736f;
  u32x4_t k[2][NJ], v[NJV];
  f32x16 dk0[1][NT], dk1[1][NT], dv[1][NTV];
  zero_acc2(dk0);
  zero_acc2(dk1);
  zero_acc2(dv);
  const int seen_from = wg_key < len ? first_query(a, wg_key, len) * a.group / RT * RT : R;
  const int per = ((R - seen_from + a.row_splits - 1) / a.row_splits + RT - 1) / RT * RT;
  const int r_first = seen_from + split * per, r_last = min(R, r_first + per);
  const int wave_first = key0 < len ? first_query(a, key0, len) * a.group : R;
  const int wave_all = key0 + 31 < len ? first_query(a, key0 + 31, len) * a.group : R;      // rows from here on see all 32 keys
  const int my_first = key < len ? first_query(a, key, len) * a.group : R;                   // rows from here on see this lane's key
  if (r_first < r_last) {
    const int kk = min(key, len - 1);
    const char* kp = reinterpret_cast<const char*>(a.k) + (b * a.k_b + kk * a.k_n + 2 * hk * a.k_h) * SZ;
    const char* vp = reinterpret_cast<const char*>(a.v) + (b * a.v_b + kk * a.v_n + hk * a.v_h) * SZ;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j) k[m][j] = load_chunk<T, VEC>(kp + m * a.k_h * SZ, 2 * j + g, a.d);
#pragma unroll
    for (int j = 0; j < NJV; ++j) v[j] = load_chunk<T, VEC>(vp, 2 * j + g, a.dv);
    typedef Stage<T, D, RT, 256, VEC> StageQ;
    typedef Stage<T, DV, RT, 256, VEC> StageO;
    StageQ sq0, sq1;
    StageO so;
    float st = 0.0f;
    const char* qp = reinterpret_cast<const char*>(a.q) + (b * a.q_b + 2 * hk * a.group * a.q_h) * SZ;
    const char* op = reinterpret_cast<const char*>(a.d_o) + o_at(a, b, 0, hk * a.group) * SZ;
    auto fetch = [&](int r0) {
      unsigned qo[StageQ::PER], oo[StageO::PER];
      const int i0 = r0 / a.group;
      row_offsets<StageQ>(a, qo, tid, r0, i0, (unsigned)a.q_n * SZ, 2u * (unsigned)a.q_h * SZ);
      row_offsets<StageO>(a, oo, tid, r0, i0, (unsigned)(a.heads * a.dv) * SZ, (unsigned)a.dv * SZ);
      const char* q = qp + i0 * a.q_n * SZ;
      sq0.load(tid, q, qo, a.d);
      sq1.load(tid, q + a.q_h * SZ, qo, a.d);
      so.load(tid, op + (long long)i0 * a.heads * a.dv * SZ, oo, a.dv);
      if (tid < 5 * RT) {
        const int w = tid >> 5, rw = min(r0 + (tid & 31), R - 1);
        if (w < 4) {
          st = (w < 2 ? a.lse : a.dots)[((long long)base * 2 + (w & 1)) * R + rw];
        } else {
          int gi;
          query_of(a, rw, gi);
          st = lam_at<T>(a, hk * a.group + gi);
        }
      }
    };
    auto place = [&](int buf) {
      sq0.store(tid, lds + buf * BUF);
      sq1.store(tid, lds + buf * BUF + QB);
      so.store(tid, lds + buf * BUF + 2 * QB);
      if (tid < 5 * RT) stat[buf][tid >> 5][tid & 31] = st;
    };
    fetch(r_first);
    place(0);
    __syncthreads();
    int cur = 0;
    for (int r0 = r_first; r0 < r_last; r0 += RT) {
      const bool more = r0 + RT < r_last;
      if (more) fetch(r0 + RT);
      if (r0 + RT > wave_first) {
        const char* buf = lds + cur * BUF;
        f32x16 p[2], dp;
        zero_acc(p);
#pragma unroll
        for (int t = 0; t < 16; ++t) dp[t] = 0.0f;
        mm_tile<T, D>(p[0], buf, 0, k[0], lane);
        mm_tile<T, D>(p[1], buf + QB, 0, k[1], lane);
        mm_tile<T, DV>(dp, buf + 2 * QB, 0, v, lane);
        const bool edge = r0 < wave_all || r0 + RT > R;
        f32x16 w[1];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 l1 = *reinterpret_cast<const f32x4*>(&stat[cur][0][8 * u + 4 * g]), l2 = *reinterpret_cast<const f32x4*>(&stat[cur][1][8 * u + 4 * g]);
          const f32x4 d1 = *reinterpret_cast<const f32x4*>(&stat[cur][2][8 * u + 4 * g]), d2 = *reinterpret_cast<const f32x4*>(&stat[cur][3][8 * u + 4 * g]);
          const f32x4 lm = *reinterpret_cast<const f32x4*>(&stat[cur][4][8 * u + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = 4 * u + e;
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[0][t], c, -l1[e])), p2 = lm[e] * __builtin_amdgcn_exp2f(__builtin_fmaf(p[1][t], c, -l2[e]));
            w[0][t] = p1 - p2;
            p[0][t] = p1 * (dp[t] - d1[e]);
            p[1][t] = p2 * (d2[e] - dp[t]);
            if (edge) {      // (the products are replaced, not the factors: nothing that stands in a hidden place gets through)
              const int row = r0 + tile_row(t, g);
              const bool seen = row >= my_first && row < R;
              w[0][t] = seen ? w[0][t] : 0.0f;
              p[0][t] = seen ? p[0][t] : 0.0f;
              p[1][t] = seen ? p[1][t] : 0.0f;
            }
          }
        }
        mm_transposed<T, DV, NTV, 1>(dv, buf + 2 * QB, 0, w, lane);
        f32x16 one[1] = {p[0]};
        mm_transposed<T, D, NT, 1>(dk0, buf, 0, one, lane);
        one[0] = p[1];
        mm_transposed<T, D, NT, 1>(dk1, buf + QB, 0, one, lane);
      }
      if (more) {
        place(cur ^ 1);
        __syncthreads();
        cur ^= 1;
      }
    }
  }
  if (key >= a.nk) return;
  const bool live = key < len;      // (rows behind the length: the clamped key's sums are not theirs)
  auto each = [&](auto put) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = live ? (m == 0 ? dk0 : dk1)[0][t][4 * u + e] * a.scale : 0.0f;
          put(m, 32 * t + 8 * u + 4 * g, x);
        }
#pragma unroll
      for (int t = 0; t < NTV; ++t) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = live ? dv[0][t][4 * u + e] : 0.0f;
        put(2, 32 * t + 8 * u + 4 * g, x);
      }
    }
  };
  const long long at = ((long long)b * a.nk + key) * a.kv_heads + hk;
  if (a.row_splits > 1) {      // [split][sample, key, head][dk1 | dk2 | dv]
    const int w = 2 * a.d + a.dv;
    float* part = a.work + ((long long)split * a.batch * a.nk * a.kv_heads + at) * w;
    each([&](int m, int col, f32x4 x) { store4<float, VEC>(part + m * a.d, col, m < 2 ? a.d : a.dv, x); });
  } else {
    T* dkp = reinterpret_cast<T*>(a.dk) + at * 2 * a.d;
    T* dvp = reinterpret_cast<T*>(a.dv_out) + at * a.dv;
    each([&](int m, int col, f32x4 x) { store4<T, VEC>(m < 2 ? dkp + m * a.d : dvp, col, m < 2 ? a.d : a.dv, x); });
  }
}

// dK, dV = the row splits' sums, in order; a thread per four elements (VEC) or one
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

// dQ of 32 rows per wave: grid (row tiles x kv_heads x batch)
template <typename T, int D, bool VEC>
__global__ __launch_bounds__(256, (D <= 64 && sizeof(T) == 2) || D <= 32 ? 2 : 1) void dq_kernel(const Args a) {
  constexpr int DV = 2 * D, KT = 32, NT = D / 32, NJ = D / (2 * Vec<T>::N), NJV = DV / (2 * Vec<T>::N), SZ = sizeof(T);
  constexpr int KB = Tile<T, D>::bytes(KT), VB = Tile<T, DV>::bytes(KT), BUF = 2 * KB + VB;
  __shared__ __align__(16) char lds[2 * BUF];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 31, g = lane >> 5;
  const int R = a.rows, tiles = (R + 127) / 128;
  int base, unit;
  grid_order(blockIdx.x, a.batch * a.kv_heads, tiles, base, unit);
  const int tile = tiles - 1 - unit;
  const int b = base / a.kv_heads, hk = base - b * a.kv_heads;
  const int len = length_of(a, b);
  const int row0 = tile * 128 + wave * 32, r = row0 + qi, rr = r < R ? r : R - 1;
  int gi;
  const int query = query_of(a, rr, gi), head = hk * a.group + gi;
  const int wg_end = end_of(a, (min(tile * 128 + 128, R) - 1) / a.group, len);
  const int my_end = r < R ? end_of(a, query, len) : 0;
  const int wave_end = row0 < R ? end_of(a, min(row0 + 31, R - 1) / a.group, len) : 0;
  const int wave_all = row0 + 31 < R ? end_of(a, row0 / a.group, len) : 0;
  const float c = a.scale * 1.44269504088896340736f;
  u32x4_t q[2][NJ], go[NJV];
  const char* qp = reinterpret_cast<const char*>(a.q) + (b * a.q_b + query * a.q_n + 2 * head * a.q_h) * SZ;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j) q[m][j] = load_chunk<T, VEC>(qp + m * a.q_h * SZ, 2 * j + g, a.d);
  const char* gp = reinterpret_cast<const char*>(a.d_o) + o_at(a, b, query, head) * SZ;
#pragma unroll
  for (int j = 0; j < NJV; ++j) go[j] = load_chunk<T, VEC>(gp, 2 * j + g, a.dv);
  const long long at = (long long)base * 2 * R + rr;
  const float l1 = a.lse[at], l2 = a.lse[at + R], d1 = a.dots[at], d2 = a.dots[at + R], lam = lam_at<T>(a, head);
  float sum2 = 0.0f;      // sum_j P_2 dP, for dlam
  f32x16 dq0[1][NT], dq1[1][NT];
  zero_acc2(dq0);
  zero_acc2(dq1);
  typedef Stage<T, D, KT, 256, VEC> StageK;
  typedef Stage<T, DV, KT, 256, VEC> StageV;
  StageK sk0, sk1;
  StageV sv;
  const char* kp = reinterpret_cast<const char*>(a.k) + (b * a.k_b + 2 * hk * a.k_h) * SZ;
  const char* vp = reinterpret_cast<const char*>(a.v) + (b * a.v_b + hk * a.v_h) * SZ;
  auto fetch = [&](int j0) {
    unsigned ko[StageK::PER], vo[StageV::PER];
    key_offsets<StageK>(ko, tid, (unsigned)a.k_n * SZ, len - 1 - j0);
    key_offsets<StageV>(vo, tid, (unsigned)a.v_n * SZ, len - 1 - j0);
    const char* k = kp + j0 * a.k_n * SZ;
    sk0.load(tid, k, ko, a.d);
    sk1.load(tid, k + a.k_h * SZ, ko, a.d);
    sv.load(tid, vp + j0 * a.v_n * SZ, vo, a.dv);
  };
  auto place = [&](char* buf) {
    sk0.store(tid, buf);
    sk1.store(tid, buf + KB);
    sv.store(tid, buf + 2 * KB);
  };
  if (wg_end > 0) {
    fetch(0);
    place(lds);
    __syncthreads();
    int cur = 0;
    for (int j0 = 0; j0 < wg_end; j0 += KT) {
      const bool more = j0 + KT < wg_end;
      if (more) fetch(j0 + KT);
      if (j0 < wave_end) {
        const char* buf = lds + cur * BUF;
        f32x16 p[2], dp;
        zero_acc(p);
#pragma unroll
        for (int t = 0; t < 16; ++t) dp[t] = 0.0f;
        mm_tile<T, D>(p[0], buf, 0, q[0], lane);
        mm_tile<T, D>(p[1], buf + KB, 0, q[1], lane);
        mm_tile<T, DV>(dp, buf + 2 * KB, 0, go, lane);
        const bool edge = j0 + KT > wave_all;
        float s = 0.0f;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[0][t], c, -l1)), p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[1][t], c, -l2));
          float both = p2 * dp[t];
          p[0][t] = p1 * (dp[t] - d1);
          p[1][t] = p2 * (d2 - dp[t]) * lam;
          if (edge) {
            const bool seen = j0 + tile_row(t, g) < my_end;
            p[0][t] = seen ? p[0][t] : 0.0f;
            p[1][t] = seen ? p[1][t] : 0.0f;
            both = seen ? both : 0.0f;
          }
          s += both;
        }
        sum2 += s;
        f32x16 one[1] = {p[0]};
        mm_transposed<T, D, NT, 1>(dq0, buf, 0, one, lane);
        one[0] = p[1];
        mm_transposed<T, D, NT, 1>(dq1, buf + KB, 0, one, lane);
      }
      if (more) {
        place(lds + (cur ^ 1) * BUF);
        __syncthreads();
        cur ^= 1;
      }
    }
  }
  sum2 += other_half(sum2);
  if (r >= R) return;
  if (g == 0) a.dots[(2LL * a.batch * a.kv_heads + base) * R + r] = sum2;
  T* out = reinterpret_cast<T*>(a.dq) + (((long long)b * a.nq + query) * a.heads + head) * 2 * a.d;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (m == 0 ? dq0 : dq1)[0][t][4 * u + e] * a.scale;
        store4<T, VEC>(out + m * a.d, 32 * t + 8 * u + 4 * g, a.d, x);
      }
}

// ---- launches: one compilation unit per element type ----------------------------------------------------------------------------------
template <typename T, int D, bool VEC>
void launch_fwd(const Args& a, hipStream_t st) {
  const int heads = a.kv_heads * a.batch;
  if (a.rows <= 32) {      // a handful of rows: one wave per workgroup, the keys split over many of them
    fwd_kernel<T, D, 1, VEC><<<a.splits * heads, 64, 0, st>>>(a);
  } else {
    fwd_kernel<T, D, 4, VEC><<<(a.rows + 127) / 128 * a.splits * heads, 256, 0, st>>>(a);
  }
  if (a.splits > 1) join_kernel<T><<<(unsigned)(((long long)heads * a.rows + 3) / 4), 256, 0, st>>>(a);
}

template <typename T, int D, bool VEC>
void launch_bwd(const Args& a, hipStream_t st) {
  const int heads = a.kv_heads * a.batch;
  rowdot_kernel<T><<<(unsigned)(((long long)heads * a.rows + 3) / 4), 256, 0, st>>>(a);
  dkv_kernel<T, D, VEC><<<(a.nk + 127) / 128 * a.row_splits * heads, 256, 0, st>>>(a);
  if (a.row_splits > 1)
    key_join_kernel<T, VEC><<<(unsigned)(((long long)heads * a.nk * (2 * a.d + a.dv) / (VEC ? 4 : 1) + 255) / 256), 256, 0, st>>>(a);
  dq_kernel<T, D, VEC><<<(a.rows + 127) / 128 * heads, 256, 0, st>>>(a);
  dlam_kernel<T><<<a.heads, 1024, 0, st>>>(a);
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
