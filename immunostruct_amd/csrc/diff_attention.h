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

template <typename T>
__device__ __forceinline__ const T* q_row(const Args& a, int b, int hk, int r, int m) {
  const int i = r / a.group, h = hk * a.group + r % a.group;
  return reinterpret_cast<const T*>(a.q) + b * a.q_b + i * a.q_n + (2 * h + m) * a.q_h;
}
template <typename T>
__device__ __forceinline__ const T* k_row(const Args& a, int b, int hk, int j, int m) {
  return reinterpret_cast<const T*>(a.k) + b * a.k_b + j * a.k_n + (2 * hk + m) * a.k_h;
}
template <typename T>
__device__ __forceinline__ const T* v_row(const Args& a, int b, int hk, int j) {
  return reinterpret_cast<const T*>(a.v) + b * a.v_b + j * a.v_n + hk * a.v_h;
}
// row r of a contiguous (batch, nq, heads, dv) tensor
__device__ __forceinline__ long long o_at(const Args& a, int b, int hk, int r) {
  return (((long long)b * a.nq + r / a.group) * a.heads + hk * a.group + r % a.group) * a.dv;
}

// ---- forward -----------------------------------------------------------------------------------------------------------------------
// grid: (row tiles x splits x kv_heads x batch), NW waves of 32 rows.  splits > 1: every workgroup takes one range of the keys and leaves
// unnormalised sums with their maxima in the workspace; join_kernel puts them together.
template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, (D <= 64 && NW > 1 ? 2 : 1)) void fwd_kernel(const Args a) {
  constexpr int DV = 2 * D, KT = 32, NT = DV / 32, NJ = D / (2 * Vec<T>::N), NTH = 64 * NW;
  constexpr int KB = Tile<T, D>::bytes(KT), VB = Tile<T, DV>::bytes(KT), BUF = 2 * KB + VB;
  __shared__ __align__(16) char lds[2 * BUF];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 31, g = lane >> 5;
  const int R = a.nq * a.group, tiles = (R + 32 * NW - 1) / (32 * NW);
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int tile = tiles - 1 - id % tiles;      // the rows that see most keys first
  id /= tiles;
  const int split = id % a.splits;
  id /= a.splits;
  const int hk = id % a.kv_heads, b = id / a.kv_heads;
  const int len = length_of(a, b);
  const int row0 = tile * 32 * NW + wave * 32, r = row0 + qi, rr = r < R ? r : R - 1;
  const int wg_last = min(tile * 32 * NW + 32 * NW, R) - 1;
  const int wg_end = end_of(a, wg_last / a.group, len);
  const int my_end = r < R ? end_of(a, rr / a.group, len) : 0;
  const int wave_end = row0 < R ? end_of(a, min(row0 + 31, R - 1) / a.group, len) : 0;      // no row of the wave sees further
  const int wave_all = row0 + 31 < R ? end_of(a, row0 / a.group, len) : 0;                  // every row of the wave sees this far
  const int per = ((wg_end + a.splits - 1) / a.splits + KT - 1) / KT * KT;
  const int first = split * per, last = min(wg_end, first + per);
  const float c = a.scale * 1.44269504088896340736f;

  u32x4_t q[2][NJ];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const T* row = q_row<T>(a, b, hk, rr, m);
#pragma unroll
    for (int j = 0; j < NJ; ++j) q[m][j] = load_chunk<T>(row, 2 * j + g, a.d, a.vec);
  }
  f32x16 o[2][NT];
  zero_acc2(o);
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

  Stage<T, D, KT, NTH> sk0, sk1;
  Stage<T, DV, KT, NTH> sv;
  auto fetch = [&](int j0) {
    sk0.load(tid, [&](int i) { return k_row<T>(a, b, hk, min(j0 + i, len - 1), 0); }, a.d, a.vec);
    sk1.load(tid, [&](int i) { return k_row<T>(a, b, hk, min(j0 + i, len - 1), 1); }, a.d, a.vec);
    sv.load(tid, [&](int i) { return v_row<T>(a, b, hk, min(j0 + i, len - 1)); }, a.dv, a.vec);
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
  const long long base = ((long long)b * a.kv_heads + hk);
  if (a.splits > 1) {
    float* w = a.work + (base * a.splits + split) * (2 * (long long)R * (a.dv + 2));
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
          store4(wm, 32 * t + 8 * u + 4 * g, a.dv, f32x4{o[m][t][4 * u], o[m][t][4 * u + 1], o[m][t][4 * u + 2], o[m][t][4 * u + 3]}, false);
    }
    return;
  }
  const float lam = lam_at<T>(a, hk * a.group + rr % a.group);
  const float w0 = total[0] != 0.0f ? 1.0f / total[0] : 0.0f, w1 = total[1] != 0.0f ? 1.0f / total[1] : 0.0f;
  if (a.lse != nullptr && g == 0) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
      a.lse[(base * 2 + m) * R + r] = total[m] != 0.0f ? __builtin_fmaf(top[m], c, __log2f(total[m])) : INFINITY;
  }
  T* out = reinterpret_cast<T*>(a.o) + o_at(a, b, hk, r);
  T* out2 = reinterpret_cast<T*>(a.o2) + o_at(a, b, hk, r);
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
      store4(out, 32 * t + 8 * u + 4 * g, a.dv, x, a.vec);
      if (a.o2 != nullptr) store4(out2, 32 * t + 8 * u + 4 * g, a.dv, y, a.vec);
    }
}

// the splits of one row put together: one wave per row, lane = column
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  const int R = a.nq * a.group, lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (long long)a.batch * a.kv_heads * R) return;
  const int r = (int)(w % R);
  const long long base = w / R;
  const int hk = (int)(base % a.kv_heads), b = (int)(base / a.kv_heads);
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
  const float lam = lam_at<T>(a, hk * a.group + r % a.group);
  T* out = reinterpret_cast<T*>(a.o) + o_at(a, b, hk, r);
  T* out2 = reinterpret_cast<T*>(a.o2) + o_at(a, b, hk, r);
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
  const int R = a.nq * a.group, lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (long long)a.batch * a.kv_heads * R) return;
  const int r = (int)(w % R);
  const long long base = w / R;
  const int hk = (int)(base % a.kv_heads), b = (int)(base / a.kv_heads);
  const long long at = o_at(a, b, hk, r);
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
    a.dots[(base * 2) * R + r] = s + lam_at<T>(a, hk * a.group + r % a.group) * s2;
    a.dots[(base * 2 + 1) * R + r] = s2;
  }
}

// dlam_h = - sum over samples and queries of D_2 (one workgroup per head, fixed order)
template <typename T>
__global__ __launch_bounds__(1024) void dlam_kernel(const Args a) {
  __shared__ float part[16];
  const int h = blockIdx.x, hk = h / a.group, gi = h % a.group, R = a.nq * a.group;
  float s = 0.0f;
  for (long long x = threadIdx.x; x < (long long)a.batch * a.nq; x += 1024) {
    const long long b = x / a.nq;
    const int i = (int)(x - b * a.nq);
    s += a.dots[((b * a.kv_heads + hk) * 2 + 1) * R + i * a.group + gi];
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

// dK, dV of 32 keys per wave: grid (key tiles x kv_heads x batch)
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void dkv_kernel(const Args a) {
  constexpr int DV = 2 * D, RT = 32, NT = D / 32, NTV = DV / 32, NJ = D / (2 * Vec<T>::N), NJV = DV / (2 * Vec<T>::N);
  constexpr int QB = Tile<T, D>::bytes(RT), OB = Tile<T, DV>::bytes(RT), BUF = 2 * QB + OB;
  __shared__ __align__(16) char lds[2 * BUF];
  __shared__ __align__(16) float stat[2][5][RT];      // lse1, lse2, D1, D2, lam of the tile's rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ki = lane & 31, g = lane >> 5;
  const int R = a.nq * a.group, tiles = (a.nk + 127) / 128;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int tile = id % tiles;      // the keys that most rows see first
  id /= tiles;
  const int hk = id % a.kv_heads, b = id / a.kv_heads;
  const int len = length_of(a, b);
  const int wg_key = tile * 128, key0 = wg_key + wave * 32, key = key0 + ki;
  const long long base = (long long)b * a.kv_heads + hk;
  const float c = a.scale * 1.44269504088896340736f;
  u32x4_t k[2][NJ], v[NJV];
  f32x16 dk0[1][NT], dk1[1][NT], dv[1][NTV];
  zero_acc2(dk0);
  zero_acc2(dk1);
  zero_acc2(dv);
  const int r_first = wg_key < len ? first_query(a, wg_key, len) * a.group / RT * RT : R;
  const int wave_first = key0 < len ? first_query(a, key0, len) * a.group : R;
  const int wave_all = key0 + 31 < len ? first_query(a, key0 + 31, len) * a.group : R;      // rows from here on see all 32 keys
  const int my_first = key < len ? first_query(a, key, len) * a.group : R;                   // rows from here on see this lane's key
  if (r_first < R) {
    const int kk = min(key, len - 1);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j) k[m][j] = load_chunk<T>(k_row<T>(a, b, hk, kk, m), 2 * j + g, a.d, a.vec);
#pragma unroll
    for (int j = 0; j < NJV; ++j) v[j] = load_chunk<T>(v_row<T>(a, b, hk, kk), 2 * j + g, a.dv, a.vec);
    Stage<T, D, RT, 256> sq0, sq1;
    Stage<T, DV, RT, 256> so;
    float st = 0.0f;
    auto fetch = [&](int r0) {
      sq0.load(tid, [&](int i) { return q_row<T>(a, b, hk, min(r0 + i, R - 1), 0); }, a.d, a.vec);
      sq1.load(tid, [&](int i) { return q_row<T>(a, b, hk, min(r0 + i, R - 1), 1); }, a.d, a.vec);
      so.load(tid, [&](int i) { return reinterpret_cast<const T*>(a.d_o) + o_at(a, b, hk, min(r0 + i, R - 1)); }, a.dv, a.vec);
      if (tid < 5 * RT) {
        const int w = tid >> 5, rw = min(r0 + (tid & 31), R - 1);
        st = w < 2 ? a.lse[(base * 2 + w) * R + rw] : w < 4 ? a.dots[(base * 2 + w - 2) * R + rw] : lam_at<T>(a, hk * a.group + rw % a.group);
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
    for (int r0 = r_first; r0 < R; r0 += RT) {
      const bool more = r0 + RT < R;
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
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[0][t], c, -l1[e])), p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[1][t], c, -l2[e]));
            w[0][t] = p1 - lm[e] * p2;
            p[0][t] = p1 * (dp[t] - d1[e]);
            p[1][t] = -lm[e] * p2 * (dp[t] - d2[e]);
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
  T* dkp = reinterpret_cast<T*>(a.dk) + ((long long)b * a.nk + key) * (2 * a.kv_heads) * a.d + (2 * hk) * (long long)a.d;
  T* dvp = reinterpret_cast<T*>(a.dv_out) + (((long long)b * a.nk + key) * a.kv_heads + hk) * a.dv;
  const bool live = key < len;      // (rows behind the length: the clamped key's sums are not theirs)
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = live ? (m == 0 ? dk0 : dk1)[0][t][4 * u + e] * a.scale : 0.0f;
        store4(dkp + m * a.d, 32 * t + 8 * u + 4 * g, a.d, x, a.vec);
      }
#pragma unroll
  for (int t = 0; t < NTV; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = live ? dv[0][t][4 * u + e] : 0.0f;
      store4(dvp, 32 * t + 8 * u + 4 * g, a.dv, x, a.vec);
    }
}

// dQ of 32 rows per wave: grid (row tiles x kv_heads x batch)
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void dq_kernel(const Args a) {
  constexpr int DV = 2 * D, KT = 32, NT = D / 32, NJ = D / (2 * Vec<T>::N), NJV = DV / (2 * Vec<T>::N);
  constexpr int KB = Tile<T, D>::bytes(KT), VB = Tile<T, DV>::bytes(KT), BUF = 2 * KB + VB;
  __shared__ __align__(16) char lds[2 * BUF];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 31, g = lane >> 5;
  const int R = a.nq * a.group, tiles = (R + 127) / 128;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int tile = tiles - 1 - id % tiles;
  id /= tiles;
  const int hk = id % a.kv_heads, b = id / a.kv_heads;
  const int len = length_of(a, b);
  const int row0 = tile * 128 + wave * 32, r = row0 + qi, rr = r < R ? r : R - 1;
  const int wg_end = end_of(a, (min(tile * 128 + 128, R) - 1) / a.group, len);
  const int my_end = r < R ? end_of(a, rr / a.group, len) : 0;
  const int wave_end = row0 < R ? end_of(a, min(row0 + 31, R - 1) / a.group, len) : 0;
  const int wave_all = row0 + 31 < R ? end_of(a, row0 / a.group, len) : 0;
  const long long base = (long long)b * a.kv_heads + hk;
  const float c = a.scale * 1.44269504088896340736f;
  u32x4_t q[2][NJ], go[NJV];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j) q[m][j] = load_chunk<T>(q_row<T>(a, b, hk, rr, m), 2 * j + g, a.d, a.vec);
#pragma unroll
  for (int j = 0; j < NJV; ++j) go[j] = load_chunk<T>(reinterpret_cast<const T*>(a.d_o) + o_at(a, b, hk, rr), 2 * j + g, a.dv, a.vec);
  const float l1 = a.lse[(base * 2) * R + rr], l2 = a.lse[(base * 2 + 1) * R + rr];
  const float d1 = a.dots[(base * 2) * R + rr], d2 = a.dots[(base * 2 + 1) * R + rr], lam = lam_at<T>(a, hk * a.group + rr % a.group);
  f32x16 dq0[1][NT], dq1[1][NT];
  zero_acc2(dq0);
  zero_acc2(dq1);
  Stage<T, D, KT, 256> sk0, sk1;
  Stage<T, DV, KT, 256> sv;
  auto fetch = [&](int j0) {
    sk0.load(tid, [&](int i) { return k_row<T>(a, b, hk, min(j0 + i, len - 1), 0); }, a.d, a.vec);
    sk1.load(tid, [&](int i) { return k_row<T>(a, b, hk, min(j0 + i, len - 1), 1); }, a.d, a.vec);
    sv.load(tid, [&](int i) { return v_row<T>(a, b, hk, min(j0 + i, len - 1)); }, a.dv, a.vec);
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
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[0][t], c, -l1)), p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[1][t], c, -l2));
          p[0][t] = p1 * (dp[t] - d1);
          p[1][t] = -lam * p2 * (dp[t] - d2);
          if (edge) {
            const bool seen = j0 + tile_row(t, g) < my_end;
            p[0][t] = seen ? p[0][t] : 0.0f;
            p[1][t] = seen ? p[1][t] : 0.0f;
          }
        }
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
  if (r >= R) return;
  const int i = r / a.group, h = hk * a.group + r % a.group;
  T* out = reinterpret_cast<T*>(a.dq) + (((long long)b * a.nq + i) * a.heads + h) * 2 * a.d;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (m == 0 ? dq0 : dq1)[0][t][4 * u + e] * a.scale;
        store4(out + m * a.d, 32 * t + 8 * u + 4 * g, a.d, x, a.vec);
      }
}

// ---- launches: one compilation unit per element type ----------------------------------------------------------------------------------
template <typename T, int D>
void launch_fwd(const Args& a, hipStream_t st) {
  const int R = a.nq * a.group;
  if (R <= 32) {      // a handful of rows: one wave per workgroup, the keys split over many of them
    fwd_kernel<T, D, 1><<<a.splits * a.kv_heads * a.batch, 64, 0, st>>>(a);
  } else {
    fwd_kernel<T, D, 4><<<(R + 127) / 128 * a.splits * a.kv_heads * a.batch, 256, 0, st>>>(a);
  }
  if (a.splits > 1) join_kernel<T><<<(unsigned)(((long long)a.batch * a.kv_heads * R + 3) / 4), 256, 0, st>>>(a);
}

template <typename T, int D>
void launch_bwd(const Args& a, hipStream_t st) {
  const int R = a.nq * a.group;
  rowdot_kernel<T><<<(unsigned)(((long long)a.batch * a.kv_heads * R + 3) / 4), 256, 0, st>>>(a);
  dlam_kernel<T><<<a.heads, 1024, 0, st>>>(a);
  dkv_kernel<T, D><<<(a.nk + 127) / 128 * a.kv_heads * a.batch, 256, 0, st>>>(a);
  dq_kernel<T, D><<<(R + 127) / 128 * a.kv_heads * a.batch, 256, 0, st>>>(a);
}

// the built width a call runs at: heads of at most D elements, values of at most 2 D (shorter rows are padded with zeros on chip);
// 0: wider than any.  32-bit inputs stop at 64 / 128: the resident operands of wider heads do not fit a wave's 512 registers.
inline int class_of(const Args& a) {
  const int need = a.d > (a.dv + 1) / 2 ? a.d : (a.dv + 1) / 2;
  return need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 && a.type != TYPE_F32 ? 128 : 0;
}

void run_f32(const Args& a, bool backward, hipStream_t st);
void run_bf16(const Args& a, bool backward, hipStream_t st);
void run_f16(const Args& a, bool backward, hipStream_t st);

}  // namespace da
}  // namespace is
