// Group norm with an activation, channels last (batch, n, channels), statistics over a sample's valid rows and a group's channels.
//
//   xhat = (x - mean) rstd,  z = xhat w + b,  y = act(z)
//   dz = dy act'(z),  dw = sum dz xhat,  db = sum dz,  t = dz w,  dx = rstd (t - mean(t) - xhat mean(t xhat))
//
// Bound by bytes: x in and y out; x, dy in and dx out.  Forms, chosen by size (plan()):
//   rows  n = 1, a group has at most 64 chunks: a group lives in neighbouring lanes, every sum is a few lane moves,
//         a workgroup walks many samples and keeps its channels' dw / db sums in registers
//         ((24320, 1, 512) bf16, 8 groups: 19 us forward, 28 + 6 backward = 2.6 / 2.7 TB/s, launch and drain included).
//         A group of any other width goes into neighbouring lanes too, whole groups to a wave ((20000, 1, 768) bf16, 32 groups of 24 channels: 24 us forward,
//         51 a backward call; as slabs of a sample a workgroup, with a record of dw / db each, 104 and 185).
//   wide  n = 1, groups of more chunks than a wave has lanes, 1024 at most: a workgroup per group, likewise over many samples
//         ((8192, 1, 4096) bf16, one group: 43 us forward, 92 backward; as row blocks 174 and 379).
//   slab  a workgroup holds all rows of one sample's slice of whole groups in registers (up to 16 chunks a thread): one read, exact two-step
//         variance, one write.  Slices are as narrow as 64-byte row segments allow, so that small batches still fill the chip
//         ((128, 190, 64) fp32, 8 groups: 6.4 us forward, 10.0 + 3.8 backward).
//   long  a sample does not fit: row blocks leave (mean, M2) / (sum t, sum t xhat) of every group, a small launch joins a sample's blocks (one
//         wave per sample and group; done by every workgroup of the next pass it cost 50 us at (2, 65536, 512), 32 groups), a third
//         writes.  Block sums are taken about each thread's own first value, so a large mean costs no precision
//         ((2, 65536, 512) bf16, 32 groups: 30 + 6 + 50 us forward, 68 + 5 + 73 + 6 backward; eight passes of 134 MB in all, 4.5 TB/s).
//         Groups of more than 256 chunks are cut into parts, which join like row blocks ((4, 2048, 4096) bf16, one group: 50 us forward, 94
//         backward; a workgroup per sample and group that re-reads took 26 and 19 ms).
// Chunks are 16 bytes where pointers, strides and the group width allow, single elements otherwise (a chunk never straddles two groups).
// dw and db: one record [2][channels] per workgroup (long: per row block where a sample has several), summed in a fixed order by a last launch.  Where there
// are more samples than the chip holds workgroups, a workgroup walks many.
#include "../../include/immunostruct_hip.h"
#include "tiles16.h"

namespace is {
namespace gn {

typedef IsGroupNorm Args;
enum Form { ROWS, WIDE, SLAB, LONG };
struct Plan {
  Form form;
  int ve;              // elements of a chunk
  int slice, slices;   // channels of a workgroup (whole groups), their number
  int per_thread;      // slab, wide: chunks a thread holds
  int blocks, rows;    // long: row blocks of a sample, rows of one; rows, wide: workgroups
  int parts;           // long: slices of a group (more than one: a slice is at most a group's part, the last one may be narrower)
  int records;         // of dw / db
  bool pow2;           // rows: groups of a power of two of 16-byte chunks
};

__device__ __forceinline__ int length_of(const Args& a, int b) {
  const int n = a.lengths != nullptr ? a.lengths[b] : a.n;
  return n < 0 ? 0 : (n > a.n ? a.n : n);
}
template <typename T>
__device__ __forceinline__ float param(const Args& a, const void* p, int c, float other) {
  if (p == nullptr) return other;
  return a.weight_type == TYPE_F32 ? reinterpret_cast<const float*>(p)[c] : (float)reinterpret_cast<const T*>(p)[c];
}
__device__ __forceinline__ float act(float z, int kind) {
  if (kind == 1) return z * rcp_f(1.0f + __expf(-z));
  if (kind == 2) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752440f));
  if (kind == 3) return z > 0.0f ? z : (z != z ? z : 0.0f);
  return z;
}
__device__ __forceinline__ float act_slope(float z, int kind) {
  if (kind == 1) {
    const float s = rcp_f(1.0f + __expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  if (kind == 2) return 0.5f * (1.0f + erff(z * 0.70710678118654752440f)) + z * 0.39894228040143267794f * __expf(-0.5f * z * z);
  if (kind == 3) return z > 0.0f ? 1.0f : 0.0f;
  return 1.0f;
}

// a chunk of VE elements (1: a single element in word 0)
template <typename T, int VE>
struct Chunk {
  float x[VE];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VE == 1) x[0] = (float)*p;
    else Vec<T>::unpack(*reinterpret_cast<const u32x4_t*>(p), x);
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VE == 1) *p = (T)x[0];
    else *reinterpret_cast<u32x4_t*>(p) = Vec<T>::pack(x);
  }
};
// the raw bits, for chunks that wait in registers
template <typename T, int VE> struct Held {
  typedef typename std::conditional<VE == 1, T, u32x4_t>::type Raw;
  Raw v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void zero() { v = Raw{}; }
  __device__ __forceinline__ void get(float (&x)[VE]) const {
    if constexpr (VE == 1) x[0] = (float)v;
    else Vec<T>::unpack(v, x);
  }
};

__device__ __forceinline__ float wave_sum(float v) {
  v = sum_over_r(v);
  return v + other_half(v);
}

// Threads of a workgroup over a slice: thread = (row lane rl, column chunk col); cols chunks side by side, rl < lanes.
struct Place {
  int cols, lanes, col, rl;
  bool on;
  __device__ __forceinline__ Place(int slice, int ve, int width) {      // width: the channels of the slice that are there
    cols = slice / ve;
    lanes = 256 / cols;
    rl = threadIdx.x / cols;
    col = threadIdx.x - rl * cols;
    on = rl < lanes && col * ve < width;
  }
};
// sum of v over a slice's group (the threads of cpg neighbouring columns and every row lane), in each of its threads.  256 floats of LDS each.
__device__ __forceinline__ float group_sum(float v, const Place& p, int cpg, float* all, float* out) {
  const int groups = p.cols / cpg, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, each = p.lanes * cpg;
  __syncthreads();
  all[threadIdx.x] = p.on ? v : 0.0f;
  __syncthreads();
  for (int g = wave; g < groups; g += 4) {
    float s = 0.0f;
    for (int i = lane; i < each; i += 64) {
      const int r = i / cpg;
      s += all[r * p.cols + g * cpg + i - r * cpg];
    }
    s = wave_sum(s);
    if (lane == 0) out[g] = s;
  }
  __syncthreads();
  return out[p.on ? p.col / cpg : 0];
}
// the channels' sums of (dz xhat, dz) over the row lanes -> record [2][channels]
template <int VE>
__device__ __forceinline__ void channel_record(const float (&sw)[VE], const float (&sb)[VE], const Place& p, float* lds, float* record, int channels, int c0, int there) {
  const int width = p.cols * VE;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    __syncthreads();
    if (p.on) {
#pragma unroll
      for (int e = 0; e < VE; ++e) lds[p.rl * width + p.col * VE + e] = m == 0 ? sw[e] : sb[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < there; c += 256) {
      float s = 0.0f;
      for (int r = 0; r < p.lanes; ++r) s += lds[r * width + c];
      record[(long long)m * channels + c0 + c] = s;
    }
  }
}

// ---- rows: n = 1 ---------------------------------------------------------------------------------------------------------------------
// POW2: cols chunk columns side by side (a group of a power of two of chunks never straddles a wave), sums by exchange.  Otherwise a wave holds as many whole
// groups as fit its lanes, the rest of them idle; cols is the number of group columns, sums go down a tree to the group's first lane and back.
template <typename T, int VE, bool POW2, bool BACK>
__global__ __launch_bounds__(256) void rows_kernel(const Args a, const int cpg, const int cols) {
  __shared__ float lds[BACK ? 256 * VE : 1];
  const int lane = threadIdx.x & 63, cg = cpg * VE;
  int lanes, rl, cl, pos;      // rows side by side, this thread's row, its chunk column, its place in the group
  bool there;                  // part of the layout
  if constexpr (POW2) {
    lanes = 256 / cols;
    rl = threadIdx.x / cols;
    cl = threadIdx.x - rl * cols;
    pos = cl & (cpg - 1);
    there = rl < lanes;
  } else {
    const int whole = 64 / cpg, slot = lane / cpg, at = (threadIdx.x >> 6) * whole + slot;
    pos = lane - slot * cpg;
    lanes = 4 * whole / cols;
    rl = at / cols;
    cl = (at - rl * cols) * cpg + pos;
    there = slot < whole && rl < lanes;
  }
  const int width = (POW2 ? cols : cols * cpg) * VE, c = blockIdx.y * width + cl * VE;
  const bool on = there && c < a.channels;
  const int cc = on ? c : 0, g = cc / cg;
  float w[VE], o[VE], sw[VE], sb[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    w[e] = param<T>(a, a.weight, cc + e, 1.0f);
    o[e] = param<T>(a, a.bias, cc + e, 0.0f);
    sw[e] = sb[e] = 0.0f;
  }
  const float inv = 1.0f / (float)cg;
  int half = 1;
  while (2 * half < cpg) half *= 2;
  auto sum = [&](float v) {      // over the group's cpg neighbouring lanes
    if constexpr (POW2) {
      for (int m = 1; m < cpg; m *= 2) v += __shfl_xor(v, m);
      return v;
    } else {
      for (int m = half; m > 0; m /= 2) {
        const float other = __shfl_down(v, m);
        v += pos + m < cpg ? other : 0.0f;
      }
      return __shfl(v, lane - pos);
    }
  };
  const int step = gridDim.x * lanes;
  for (int b0 = blockIdx.x * lanes; b0 < a.batch; b0 += step) {      // uniform: every lane takes part in the lane moves
    const int b = b0 + rl;
    const bool live = on && b < a.batch && length_of(a, b < a.batch ? b : 0) > 0;
    Chunk<T, VE> x, d;
#pragma unroll
    for (int e = 0; e < VE; ++e) x.x[e] = d.x[e] = 0.0f;
    if (live) x.load(reinterpret_cast<const T*>(a.x) + b * a.x_b + c);
    if constexpr (BACK) {
      if (live) d.load(reinterpret_cast<const T*>(a.dy) + (long long)b * a.channels + c);
    }
    if constexpr (!BACK) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < VE; ++e) s += x.x[e];
      const float mean = sum(s) * inv;
      s = 0.0f;
#pragma unroll
      for (int e = 0; e < VE; ++e) s += (x.x[e] - mean) * (x.x[e] - mean);
      const float rstd = 1.0f / sqrtf(sum(s) * inv + a.eps);
      if (on && b < a.batch) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x.x[e] = live ? act((x.x[e] - mean) * rstd * w[e] + o[e], a.activation) : 0.0f;
        x.store(reinterpret_cast<T*>(a.y) + (long long)b * a.channels + c);
        if (pos == 0) {
          float* st = a.stats + 2 * ((long long)b * a.groups + g);
          st[0] = mean;
          st[1] = rstd;
        }
      }
    } else {
      float mean = 0.0f, rstd = 0.0f;
      if (live) {
        const float* st = a.stats + 2 * ((long long)b * a.groups + g);
        mean = st[0];
        rstd = st[1];
      }
      float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float hat = (x.x[e] - mean) * rstd;
        const float dz = live ? d.x[e] * act_slope(hat * w[e] + o[e], a.activation) : 0.0f;
        sw[e] += dz * hat;
        sb[e] += dz;
        x.x[e] = hat;
        d.x[e] = dz * w[e];
        t1 += d.x[e];
        t2 += d.x[e] * hat;
      }
      t1 = sum(t1) * inv;
      t2 = sum(t2) * inv;
      if (on && b < a.batch && a.dx != nullptr) {
#pragma unroll
        for (int e = 0; e < VE; ++e) d.x[e] = live ? rstd * (d.x[e] - t1 - x.x[e] * t2) : 0.0f;
        d.store(reinterpret_cast<T*>(a.dx) + (long long)b * a.channels + c);
      }
    }
  }
  if constexpr (BACK) {
    if (a.dweight != nullptr) {
      const int c0 = blockIdx.y * width;
      float* record = a.work + (long long)blockIdx.x * 2 * a.channels;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        __syncthreads();
        if (there) {
#pragma unroll
          for (int e = 0; e < VE; ++e) lds[rl * width + cl * VE + e] = m == 0 ? sw[e] : sb[e];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < width && c0 + i < a.channels; i += 256) {
          float s = 0.0f;
          for (int r = 0; r < lanes; ++r) s += lds[r * width + i];
          record[(long long)m * a.channels + c0 + i] = s;
        }
      }
    }
  }
}

// ---- wide: n = 1, a workgroup per group -----------------------------------------------------------------------------------------------
template <typename T, int VE, int K, bool BACK>
__global__ __launch_bounds__(256) void wide_kernel(const Args a) {
  __shared__ float scratch[2][2][4];
  const int g = blockIdx.y, cg = a.channels / a.groups, tid = threadIdx.x, c = g * cg + tid * VE;
  bool on[K];
  float w[K][VE], o[K][VE], sw[K][VE], sb[K][VE];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    on[k] = (tid + k * 256) * VE < cg;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      w[k][e] = on[k] ? param<T>(a, a.weight, c + k * 256 * VE + e, 1.0f) : 0.0f;
      o[k][e] = on[k] ? param<T>(a, a.bias, c + k * 256 * VE + e, 0.0f) : 0.0f;
      sw[k][e] = sb[k][e] = 0.0f;
    }
  }
  const float inv = 1.0f / (float)cg;
  auto sums = [&](float (&v)[2], float (&lds)[2][4]) {      // over the workgroup, in every thread
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      v[m] = wave_sum(v[m]);
      if ((tid & 63) == 0) lds[m][tid >> 6] = v[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m) v[m] = (lds[m][0] + lds[m][1]) + (lds[m][2] + lds[m][3]);
  };
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {      // (uniform: every barrier is met)
    const bool live = length_of(a, b) > 0;
    Chunk<T, VE> x[K], d[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < VE; ++e) x[k].x[e] = d[k].x[e] = 0.0f;
      if (live && on[k]) {
        x[k].load(reinterpret_cast<const T*>(a.x) + b * a.x_b + c + k * 256 * VE);
        if constexpr (BACK) d[k].load(reinterpret_cast<const T*>(a.dy) + (long long)b * a.channels + c + k * 256 * VE);
      }
    }
    float* st = a.stats + 2 * ((long long)b * a.groups + g);
    if constexpr (!BACK) {
      float s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < VE; ++e) s[0] += x[k].x[e];
      sums(s, scratch[0]);
      const float mean = s[0] * inv;
      s[0] = s[1] = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float off = on[k] ? x[k].x[e] - mean : 0.0f;
          s[0] += off * off;
        }
      sums(s, scratch[1]);      // (the next sample's first sums use the other half: its readers are past this barrier)
      const float rstd = 1.0f / sqrtf(s[0] * inv + a.eps);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[k].x[e] = live ? act((x[k].x[e] - mean) * rstd * w[k][e] + o[k][e], a.activation) : 0.0f;
        if (on[k]) x[k].store(reinterpret_cast<T*>(a.y) + (long long)b * a.channels + c + k * 256 * VE);
      }
      if (tid == 0) {
        st[0] = mean;
        st[1] = rstd;
      }
    } else {
      const float mean = live ? st[0] : 0.0f, rstd = live ? st[1] : 0.0f;
      float t[2] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float hat = (x[k].x[e] - mean) * rstd;
          const float dz = live && on[k] ? d[k].x[e] * act_slope(hat * w[k][e] + o[k][e], a.activation) : 0.0f;
          sw[k][e] += dz * hat;
          sb[k][e] += dz;
          x[k].x[e] = hat;
          d[k].x[e] = dz * w[k][e];
          t[0] += d[k].x[e];
          t[1] += d[k].x[e] * hat;
        }
      sums(t, scratch[(b / gridDim.x) & 1]);      // (halves in turn: a sample's writers have passed the barrier behind the last readers of theirs)
      t[0] *= inv;
      t[1] *= inv;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < VE; ++e) d[k].x[e] = live ? rstd * (d[k].x[e] - t[0] - x[k].x[e] * t[1]) : 0.0f;
        if (on[k] && a.dx != nullptr) d[k].store(reinterpret_cast<T*>(a.dx) + (long long)b * a.channels + c + k * 256 * VE);
      }
    }
  }
  if constexpr (BACK) {
    if (a.dweight != nullptr) {
      float* record = a.work + (long long)blockIdx.x * 2 * a.channels + c;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (on[k]) {
            record[k * 256 * VE + e] = sw[k][e];
            record[a.channels + k * 256 * VE + e] = sb[k][e];
          }
    }
  }
}

// ---- slab: a sample's slice in registers ------------------------------------------------------------------------------------------------
template <typename T, int VE, int K>
__global__ __launch_bounds__(256) void slab_fwd_kernel(const Args a, const int slice) {
  __shared__ float all[256], out[256];
  const int slices = a.channels / slice, b = blockIdx.x / slices, c0 = (blockIdx.x - b * slices) * slice, cg = a.channels / a.groups;
  const int len = length_of(a, b), cpg = cg / VE;
  const Place p(slice, VE, slice);
  const int c = c0 + p.col * VE;
  const T* x = reinterpret_cast<const T*>(a.x) + b * a.x_b + c;
  T* y = reinterpret_cast<T*>(a.y) + (long long)b * a.n * a.channels + c;
  Held<T, VE> h[K];
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int row = p.rl + k * p.lanes;
    h[k].zero();
    if (p.on && row < len) h[k].load(x + row * a.x_n);
  }
  float w[VE], o[VE], v[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    w[e] = p.on ? param<T>(a, a.weight, c + e, 1.0f) : 0.0f;
    o[e] = p.on ? param<T>(a, a.bias, c + e, 0.0f) : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    h[k].get(v);
#pragma unroll
    for (int e = 0; e < VE; ++e) s += v[e];
  }
  const float inv = 1.0f / ((float)(len > 0 ? len : 1) * (float)cg);
  const float mean = group_sum(s, p, cpg, all, out) * inv;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (p.rl + k * p.lanes < len) {
      h[k].get(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) s += (v[e] - mean) * (v[e] - mean);
    }
  const float rstd = 1.0f / sqrtf(group_sum(s, p, cpg, all, out) * inv + a.eps);
  if (!p.on) return;
  if (p.rl == 0 && p.col % cpg == 0) {
    float* st = a.stats + 2 * ((long long)b * a.groups + c / cg);
    st[0] = mean;
    st[1] = rstd;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int row = p.rl + k * p.lanes;
    if (row < a.n) {
      Chunk<T, VE> r;
      h[k].get(r.x);
#pragma unroll
      for (int e = 0; e < VE; ++e) r.x[e] = row < len ? act((r.x[e] - mean) * rstd * w[e] + o[e], a.activation) : 0.0f;
      r.store(y + (long long)row * a.channels);
    }
  }
}

// WALK: a workgroup walks the samples blockIdx.x / slices, + gridDim.x / slices, ...; without it there is one for every sample
template <typename T, int VE, int K, bool WALK>
__global__ __launch_bounds__(256) void slab_bwd_kernel(const Args a, const int slice) {
  __shared__ float all[256], out[256], lds[256 * VE];
  const int slices = a.channels / slice, b0 = blockIdx.x / slices, step = gridDim.x / slices, c0 = (blockIdx.x - b0 * slices) * slice, cg = a.channels / a.groups;
  const int cpg = cg / VE;
  const Place p(slice, VE, slice);
  const int c = c0 + p.col * VE;
  float tw[VE], tb[VE];      // over the workgroup's samples
#pragma unroll
  for (int e = 0; e < VE; ++e) tw[e] = tb[e] = 0.0f;
  for (int b = b0; b < a.batch; b += step) {      // (uniform: every barrier is met)
    const int len = length_of(a, b);
    const T* x = reinterpret_cast<const T*>(a.x) + b * a.x_b + c;
    const long long at = (long long)b * a.n * a.channels + c;
    const T* dy = reinterpret_cast<const T*>(a.dy) + at;
    T* dx = reinterpret_cast<T*>(a.dx) + at;
    Held<T, VE> h[K], d[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int row = p.rl + k * p.lanes;
      h[k].zero();
      d[k].zero();
      if (p.on && row < len) {
        h[k].load(x + row * a.x_n);
        d[k].load(dy + (long long)row * a.channels);
      }
    }
    float w[VE], o[VE], sw[VE], sb[VE], v[VE], u[VE];
    float mean = 0.0f, rstd = 0.0f;
    if (p.on) {
      const float* st = a.stats + 2 * ((long long)b * a.groups + c / cg);
      mean = st[0];
      rstd = st[1];
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      w[e] = p.on ? param<T>(a, a.weight, c + e, 1.0f) : 0.0f;
      o[e] = p.on ? param<T>(a, a.bias, c + e, 0.0f) : 0.0f;
      sw[e] = sb[e] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (p.rl + k * p.lanes < len) {
        h[k].get(v);
        d[k].get(u);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float hat = (v[e] - mean) * rstd, dz = u[e] * act_slope(hat * w[e] + o[e], a.activation);
          sw[e] += dz * hat;
          sb[e] += dz;
        }
      }
    float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      t1 += sb[e] * w[e];
      t2 += sw[e] * w[e];
      tw[e] += sw[e];
      tb[e] += sb[e];
    }
    const float inv = 1.0f / ((float)(len > 0 ? len : 1) * (float)cg);
    t1 = group_sum(t1, p, cpg, all, out) * inv;
    t2 = group_sum(t2, p, cpg, all, out) * inv;
    if (p.on && a.dx != nullptr) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int row = p.rl + k * p.lanes;
        if (row < a.n) {
          Chunk<T, VE> r;
          h[k].get(v);
          d[k].get(u);
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float hat = (v[e] - mean) * rstd, dz = u[e] * act_slope(hat * w[e] + o[e], a.activation);
            r.x[e] = row < len ? rstd * (dz * w[e] - t1 - hat * t2) : 0.0f;
          }
          r.store(dx + (long long)row * a.channels);
        }
      }
    }
    if constexpr (!WALK) break;
  }
  if (a.dweight != nullptr) channel_record<VE>(tw, tb, p, lds, a.work + (long long)b0 * 2 * a.channels, a.channels, c0, slice);
}

// ---- long: row blocks ---------------------------------------------------------------------------------------------------------------------
// workspace: pairs[sample][group][block][part][2], joined[sample][group][2], then the dw / db records.  Workgroup = (sample, block, slice); the
// backward's first pass walks every records / blocks-th sample where there are many, so that the records stay few
struct Block {
  int b, block, part, c0, width, first, last, len;
  __device__ __forceinline__ Block(const Args& a, const Plan& p) {
    const int slices = p.slices, cg = a.channels / a.groups;
    int id = blockIdx.x;
    const int s = id % slices;
    part = s % p.parts;
    c0 = p.parts == 1 ? s * p.slice : s / p.parts * cg + part * p.slice;
    width = p.parts == 1 ? p.slice : min(p.slice, cg - part * p.slice);
    id /= slices;
    block = id % p.blocks;
    first = block * p.rows;
    at(a, p, id / p.blocks);
  }
  __device__ __forceinline__ void at(const Args& a, const Plan& p, int sample) {
    b = sample;
    len = sample < a.batch ? length_of(a, sample) : 0;
    last = min(first + p.rows, len);
  }
};

__device__ __forceinline__ float* pair_at(const Args& a, const Plan& plan, const Block& k, int group) {
  return a.work + 2 * ((((long long)k.b * a.groups + group) * plan.blocks + k.block) * plan.parts + k.part);
}

// rows first, first + step ... below end, four at a time: all loads of a batch are in flight before its first use
constexpr int BATCH = 4;
template <typename H, typename LoadF, typename UseF>
__device__ __forceinline__ void batches(int first, int end, int step, LoadF load, UseF use) {
  for (int row = first; row < end; row += BATCH * step) {
    H h[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (row + u * step < end) load(row + u * step, h[u]);
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (row + u * step < end) use(row + u * step, h[u]);
  }
}
template <typename T, int VE>
struct Pair {
  Held<T, VE> x, d;
};

template <typename T, int VE>
__global__ __launch_bounds__(256) void long_stat_kernel(const Args a, const Plan plan) {
  __shared__ float all[256], out[256];
  const Block k(a, plan);
  const int cg = a.channels / a.groups, share = plan.parts == 1 ? cg : k.width, cpg = (plan.parts == 1 ? cg : plan.slice) / VE;
  const Place p(plan.slice, VE, k.width);
  const int c = k.c0 + p.col * VE;
  float s[VE], q[VE], base[VE];
  int count = 0;
#pragma unroll
  for (int e = 0; e < VE; ++e) s[e] = q[e] = base[e] = 0.0f;
  if (p.on) {
    const T* x = reinterpret_cast<const T*>(a.x) + k.b * a.x_b + c;
    Chunk<T, VE> v;
    int row = k.first + p.rl;
    if (row < k.last) {
      v.load(x + row * a.x_n);
#pragma unroll
      for (int e = 0; e < VE; ++e) base[e] = v.x[e];
      ++count;
    }
    batches<Held<T, VE>>(row + p.lanes, k.last, p.lanes, [&](int r, Held<T, VE>& h) { h.load(x + r * a.x_n); }, [&](int, const Held<T, VE>& h) {
      h.get(v.x);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float t = v.x[e] - base[e];
        s[e] += t;
        q[e] += t * t;
      }
      ++count;
    });
  }
  const float rows = (float)(k.last > k.first ? k.last - k.first : 0), total = rows * (float)share;
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < VE; ++e) sum += (float)count * base[e] + s[e];
  const float mean = group_sum(sum, p, cpg, all, out) / (total > 0.0f ? total : 1.0f);
  float m2 = 0.0f;
  if (count > 0) {
    const float n = (float)count;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float off = s[e] / n, far = base[e] + off - mean;      // this thread's channel mean about its base, and about the block's mean
      m2 += (q[e] - s[e] * off) + n * far * far;
    }
  }
  m2 = group_sum(m2, p, cpg, all, out);
  if (p.on && p.rl == 0 && p.col % cpg == 0) {
    float* at = pair_at(a, plan, k, c / cg);
    at[0] = mean;
    at[1] = m2;
  }
}

// one wave per (sample, group): forward -> mean and rstd; backward -> the means of t and t xhat
template <bool BACK>
__global__ __launch_bounds__(256) void long_join_kernel(const Args a, const Plan plan) {
  const int lane = threadIdx.x & 63, cg = a.channels / a.groups, entries = plan.blocks * plan.parts;
  const long long all = (long long)a.batch * a.groups;
  for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < all; i += gridDim.x * 4LL) {
    const int len = length_of(a, (int)(i / a.groups));
    const float2* at = reinterpret_cast<const float2*>(a.work) + i * entries;
    const float total = (float)(len > 0 ? len : 1) * (float)cg;
    auto count = [&](int n) {      // elements behind entry n
      const int block = n / plan.parts, part = n - block * plan.parts, width = plan.parts == 1 ? cg : min(plan.slice, cg - part * plan.slice);
      return (float)max(min((block + 1) * plan.rows, len) - block * plan.rows, 0) * (float)width;
    };
    float s0 = 0.0f, s1 = 0.0f;
    for (int n = lane; n < entries; n += 64) {
      const float2 x = at[n];
      if constexpr (BACK) {
        s0 += x.x;
        s1 += x.y;
      } else {
        s0 += x.x * (count(n) / total);
      }
    }
    s0 = wave_sum(s0);
    if constexpr (BACK) {
      s1 = wave_sum(s1);
      if (lane == 0) reinterpret_cast<float2*>(a.work)[all * entries + i] = make_float2(s0 / total, s1 / total);
    } else {
      for (int n = lane; n < entries; n += 64) {
        const float2 x = at[n];
        const float off = x.x - s0;
        s1 += x.y + count(n) * off * off;
      }
      s1 = wave_sum(s1);
      if (lane == 0) reinterpret_cast<float2*>(a.stats)[i] = make_float2(s0, 1.0f / sqrtf(s1 / total + a.eps));
    }
  }
}

template <typename T, int VE>
__global__ __launch_bounds__(256) void long_apply_kernel(const Args a, const Plan plan) {
  const Block k(a, plan);
  const int cg = a.channels / a.groups;
  const Place p(plan.slice, VE, k.width);
  if (!p.on) return;
  const int c = k.c0 + p.col * VE;
  const float* st = a.stats + 2 * ((long long)k.b * a.groups + c / cg);
  const float mean = st[0], rstd = st[1];
  float w[VE], o[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    w[e] = param<T>(a, a.weight, c + e, 1.0f);
    o[e] = param<T>(a, a.bias, c + e, 0.0f);
  }
  const T* x = reinterpret_cast<const T*>(a.x) + k.b * a.x_b + c;
  T* y = reinterpret_cast<T*>(a.y) + (long long)k.b * a.n * a.channels + c;
  const int end = min(k.first + plan.rows, a.n);
  batches<Held<T, VE>>(k.first + p.rl, end, p.lanes, [&](int row, Held<T, VE>& h) {
    h.zero();
    if (row < k.len) h.load(x + row * a.x_n);
  }, [&](int row, const Held<T, VE>& h) {
    Chunk<T, VE> v;
    h.get(v.x);
#pragma unroll
    for (int e = 0; e < VE; ++e) v.x[e] = row < k.len ? act((v.x[e] - mean) * rstd * w[e] + o[e], a.activation) : 0.0f;
    v.store(y + (long long)row * a.channels);
  });
}

template <typename T, int VE, bool WALK>
__global__ __launch_bounds__(256) void long_sum_kernel(const Args a, const Plan plan) {
  __shared__ float all[256], out[256], lds[256 * VE];
  Block k(a, plan);
  const int cg = a.channels / a.groups, cpg = (plan.parts == 1 ? cg : plan.slice) / VE;
  const Place p(plan.slice, VE, k.width);
  const int c = k.c0 + p.col * VE, step = plan.records / plan.blocks;
  const long long pairs = 2LL * a.batch * (plan.blocks * plan.parts + 1) * a.groups, index = (long long)k.b * plan.blocks + k.block;
  float w[VE], o[VE], tw[VE], tb[VE];      // tw, tb: over the workgroup's samples
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    w[e] = p.on ? param<T>(a, a.weight, c + e, 1.0f) : 0.0f;
    o[e] = p.on ? param<T>(a, a.bias, c + e, 0.0f) : 0.0f;
    tw[e] = tb[e] = 0.0f;
  }
  for (; k.b < a.batch; k.at(a, plan, k.b + step)) {      // (uniform: every barrier is met)
    float sw[VE], sb[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) sw[e] = sb[e] = 0.0f;
    if (p.on) {
      const float* st = a.stats + 2 * ((long long)k.b * a.groups + c / cg);
      const float mean = st[0], rstd = st[1];
      const T* x = reinterpret_cast<const T*>(a.x) + k.b * a.x_b + c;
      const T* dy = reinterpret_cast<const T*>(a.dy) + (long long)k.b * a.n * a.channels + c;
      batches<Pair<T, VE>>(k.first + p.rl, k.last, p.lanes, [&](int row, Pair<T, VE>& h) {
        h.x.load(x + row * a.x_n);
        h.d.load(dy + (long long)row * a.channels);
      }, [&](int, const Pair<T, VE>& h) {
        float v[VE], d[VE];
        h.x.get(v);
        h.d.get(d);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float hat = (v[e] - mean) * rstd, dz = d[e] * act_slope(hat * w[e] + o[e], a.activation);
          sw[e] += dz * hat;
          sb[e] += dz;
        }
      });
    }
    float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      t1 += sb[e] * w[e];
      t2 += sw[e] * w[e];
      tw[e] += sw[e];
      tb[e] += sb[e];
    }
    t1 = group_sum(t1, p, cpg, all, out);
    t2 = group_sum(t2, p, cpg, all, out);
    if (p.on && p.rl == 0 && p.col % cpg == 0) {
      float* at = pair_at(a, plan, k, c / cg);
      at[0] = t1;
      at[1] = t2;
    }
    if constexpr (!WALK) break;
  }
  if (a.dweight != nullptr) channel_record<VE>(tw, tb, p, lds, a.work + pairs + index * 2 * a.channels, a.channels, k.c0, k.width);
}

template <typename T, int VE>
__global__ __launch_bounds__(256) void long_dx_kernel(const Args a, const Plan plan) {
  const Block k(a, plan);
  const int cg = a.channels / a.groups;
  const Place p(plan.slice, VE, k.width);
  if (!p.on) return;
  const int c = k.c0 + p.col * VE;
  const float* joined = a.work + 2LL * a.batch * a.groups * plan.blocks * plan.parts + 2 * ((long long)k.b * a.groups + c / cg);
  const float t1 = joined[0], t2 = joined[1];
  const float* st = a.stats + 2 * ((long long)k.b * a.groups + c / cg);
  const float mean = st[0], rstd = st[1];
  float w[VE], o[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    w[e] = param<T>(a, a.weight, c + e, 1.0f);
    o[e] = param<T>(a, a.bias, c + e, 0.0f);
  }
  const T* x = reinterpret_cast<const T*>(a.x) + k.b * a.x_b + c;
  const long long at = (long long)k.b * a.n * a.channels + c;
  const T* dy = reinterpret_cast<const T*>(a.dy) + at;
  T* dx = reinterpret_cast<T*>(a.dx) + at;
  const int end = min(k.first + plan.rows, a.n);
  batches<Pair<T, VE>>(k.first + p.rl, end, p.lanes, [&](int row, Pair<T, VE>& h) {
    h.x.zero();
    h.d.zero();
    if (row < k.len) {
      h.x.load(x + row * a.x_n);
      h.d.load(dy + (long long)row * a.channels);
    }
  }, [&](int row, const Pair<T, VE>& h) {
    float v[VE];
    Chunk<T, VE> d;
    h.x.get(v);
    h.d.get(d.x);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float hat = (v[e] - mean) * rstd, dz = d.x[e] * act_slope(hat * w[e] + o[e], a.activation);
      d.x[e] = row < k.len ? rstd * (dz * w[e] - t1 - hat * t2) : 0.0f;
    }
    d.store(dx + (long long)row * a.channels);
  });
}

// dweight, dbias = the sums of `records` records [2][channels]: 16 columns x 64 record lanes a workgroup, then the lanes in order
template <typename T>
__global__ __launch_bounds__(1024) void param_grad_kernel(const Args a, const float* part, int records) {
  __shared__ float sum[64][17];
  const int col = threadIdx.x & 15, r0 = threadIdx.x >> 4, i = blockIdx.x * 16 + col, total = 2 * a.channels;
  float s = 0.0f;
  if (i < total) {
#pragma unroll 4
    for (int r = r0; r < records; r += 64) s += part[(long long)r * total + i];
  }
  sum[r0][col] = s;
  __syncthreads();
#pragma unroll
  for (int h = 32; h > 0; h >>= 1) {
    if (r0 < h) sum[r0][col] += sum[r0 + h][col];
    __syncthreads();
  }
  if (r0 == 0 && i < total) {
    void* out = i < a.channels ? a.dweight : a.dbias;
    const int c = i < a.channels ? i : i - a.channels;
    if (a.weight_type == TYPE_F32) reinterpret_cast<float*>(out)[c] = sum[0][col];
    else reinterpret_cast<T*>(out)[c] = (T)sum[0][col];
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
constexpr unsigned LAUNCH = 1u << 23;      // workgroups: a launch of 2^32 threads (2^24 workgroups) and more runs short of them without an error

bool sizes_ok(const Args& a) {
  return a.batch >= 1 && a.n >= 1 && a.channels >= 1 && a.groups >= 1 && a.channels % a.groups == 0 && a.channels <= (1 << 24) && a.n <= (1 << 30) &&
         (long long)a.batch * a.groups <= 0x3fffffffLL && a.type >= TYPE_F32 && a.type <= TYPE_F16;
}

// Samples that a backward pass works on at a time, each workgroup walking its share of them: bounds the records of dw and db (8 bytes a channel each).
// 2048 workgroups, 8 a CU, are as many as the chip holds.  The long form walks from there on: (8192, 2, 4112) bf16, 2 groups 313 us instead of 507 with a record
// a sample, (2500, 3000, 64), 8 groups 958 for 965.  The slab form's loop costs registers ((8192, 17, 512), 8 groups 344 for 240): it walks only beyond 64 MB
// of records, and with 32 rows or more, where they are at most 1 / 8 of x in 16 bits, not at all.
int walkers(const Args& a, int slices, bool slab) {
  long long most = 2048 / slices > 1 ? 2048 / slices : 1;
  if (slab) most = a.n >= 32 ? a.batch : most > (1 << 23) / a.channels ? most : (1 << 23) / a.channels;
  return (int)(a.batch < most ? a.batch : most);
}

// The form of a call, by sizes and alignment alone (dy, y and dx are contiguous; their pointers do not enter: x's alignment decides, and the
// library's callers allocate theirs 16-byte aligned -- checked in run()).
Plan plan(const Args& a) {
  Plan p = {};
  const int full = a.type == TYPE_F32 ? 4 : 8, size = a.type == TYPE_F32 ? 4 : 2, cg = a.channels / a.groups;
  const bool chunks = (a.x_b | a.x_n) % full == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && cg % full == 0;
  p.ve = chunks ? full : 1;
  const int cpg = cg / p.ve;
  if (a.n == 1 && cpg <= 64) {
    p.form = ROWS;
    p.pow2 = chunks && (cpg & (cpg - 1)) == 0;
    const int whole = 4 * (64 / cpg), all = p.pow2 ? a.channels / p.ve : a.groups, side = p.pow2 ? 256 : whole;      // columns: chunks or groups
    const int lanes_of = all < side ? all : side, per_pass = side / lanes_of, columns = (all + lanes_of - 1) / lanes_of;
    const long long passes = ((long long)a.batch + per_pass - 1) / per_pass;
    const long long most = 2048 / columns > 1 ? 2048 / columns : 1;      // 8 workgroups a CU
    p.blocks = (int)(passes < most ? passes : most);
    p.slice = lanes_of;
    p.slices = columns;
    p.records = p.blocks;
    if (columns <= 32768) return p;      // (the grid's second dimension)
  }
  if (a.n == 1 && cpg > 64 && cpg <= 1024 && a.groups <= 32768) {      // (groups: the grid's second dimension)
    p.form = WIDE;
    p.per_thread = cpg <= 256 ? 1 : cpg <= 512 ? 2 : 4;
    const int most = 1024 / a.groups > 1 ? 1024 / a.groups : 1;      // 4 workgroups a CU
    p.blocks = a.batch < most ? a.batch : most;
    p.slices = a.groups;
    p.records = p.blocks;
    return p;
  }
  // slices of whole groups: 64 bytes of a row at least, more while that still leaves 1024 workgroups, 256 chunks at most
  auto fits = [&](int gs) { return (long long)gs * cpg <= 256; };
  int gs = 1;
  p.parts = (cpg + 255) / 256;
  for (int k = 1; k <= a.groups && p.parts == 1; ++k) {
    if (!fits(k)) break;
    if (a.groups % k != 0) continue;
    const bool narrow = (long long)gs * cg * size < 64, many = (long long)a.batch * (a.groups / k) >= 1024;
    if (k > gs && (narrow || many)) {
      const int lanes = 256 / (k * cpg);
      if (!narrow && (long long)lanes * 16 < a.n) break;      // wider would no longer fit a workgroup's registers
      gs = k;
    }
  }
  const int lanes = p.parts == 1 ? 256 / (gs * cpg) : 0, need = p.parts == 1 ? (a.n + lanes - 1) / lanes : 0;
  if (p.parts == 1 && need <= 16) {
    p.slice = gs * cg;
    p.slices = a.groups / gs;
    p.form = SLAB;
    p.per_thread = need <= 1 ? 1 : need <= 4 ? 4 : 16;
    p.records = walkers(a, p.slices, true);
    return p;
  }
  p.form = LONG;
  // rows as wide as 256 chunks allow; 1024 workgroups, 16 rows a thread at least
  for (int k = 1; k <= a.groups && fits(k); ++k)
    if (a.groups % k == 0) gs = k;
  p.slice = p.parts == 1 ? gs * cg : (cpg + p.parts - 1) / p.parts * p.ve;
  p.slices = a.groups / gs * p.parts;
  const int per = 256 / (p.slice / p.ve) * 16;
  const long long want = 1024 / ((long long)a.batch * p.slices) > 1 ? 1024 / ((long long)a.batch * p.slices) : 1, most = (a.n + per - 1) / per;
  const int blocks = (int)(want < most ? want : most);
  p.rows = (a.n + blocks - 1) / blocks;
  p.blocks = (a.n + p.rows - 1) / p.rows;
  p.records = (p.blocks > 1 ? a.batch : walkers(a, p.slices, false)) * p.blocks;      // (row blocks: a batch of fewer than 1024 workgroups)
  return p;
}

long long work_floats(const Args& a, const Plan& p, bool backward) {
  const long long pairs = p.form == LONG ? 2LL * a.batch * (p.blocks * p.parts + 1) * a.groups : 0;
  return pairs + (backward && a.weight != nullptr ? 2LL * p.records * a.channels : 0);
}

// the samples [first, first + count) of a call (slab form)
template <typename T>
Args samples(Args a, int first, int count) {
  const long long at = (long long)first * a.n * a.channels * (long long)sizeof(T);
  auto shift = [&](const void* p, long long bytes) { return p != nullptr ? static_cast<const char*>(p) + bytes : nullptr; };
  a.x = shift(a.x, first * a.x_b * (long long)sizeof(T));
  a.y = const_cast<char*>(shift(a.y, at));
  a.dy = shift(a.dy, at);
  a.dx = const_cast<char*>(shift(a.dx, at));
  a.stats += 2LL * first * a.groups;
  if (a.lengths != nullptr) a.lengths += first;
  if (a.work != nullptr) a.work += 2LL * first * a.channels;
  a.batch = count;
  return a;
}

template <typename T, int VE>
void launch_slab(const Args& a, const Plan& p, bool backward, hipStream_t st) {
  const unsigned grid = (unsigned)((long long)a.batch * p.slices), walking = (unsigned)((long long)p.records * p.slices);
  if (backward && p.records < a.batch) {
    if (p.per_thread == 1) slab_bwd_kernel<T, VE, 1, true><<<walking, 256, 0, st>>>(a, p.slice);
    else if (p.per_thread == 4) slab_bwd_kernel<T, VE, 4, true><<<walking, 256, 0, st>>>(a, p.slice);
    else slab_bwd_kernel<T, VE, 16, true><<<walking, 256, 0, st>>>(a, p.slice);
  } else if (backward) {
    if (p.per_thread == 1) slab_bwd_kernel<T, VE, 1, false><<<grid, 256, 0, st>>>(a, p.slice);
    else if (p.per_thread == 4) slab_bwd_kernel<T, VE, 4, false><<<grid, 256, 0, st>>>(a, p.slice);
    else slab_bwd_kernel<T, VE, 16, false><<<grid, 256, 0, st>>>(a, p.slice);
  } else {
    if (p.per_thread == 1) slab_fwd_kernel<T, VE, 1><<<grid, 256, 0, st>>>(a, p.slice);
    else if (p.per_thread == 4) slab_fwd_kernel<T, VE, 4><<<grid, 256, 0, st>>>(a, p.slice);
    else slab_fwd_kernel<T, VE, 16><<<grid, 256, 0, st>>>(a, p.slice);
  }
}

template <typename T, int VE, bool POW2>
void launch_rows(const Args& a, const Plan& p, bool backward, hipStream_t st) {
  const int cpg = a.channels / a.groups / VE;
  const dim3 grid(p.blocks, p.slices);
  if (backward) rows_kernel<T, VE, POW2, true><<<grid, 256, 0, st>>>(a, cpg, p.slice);
  else rows_kernel<T, VE, POW2, false><<<grid, 256, 0, st>>>(a, cpg, p.slice);
}

template <typename T, int VE, int K>
void launch_wide(const Args& a, const Plan& p, bool backward, hipStream_t st) {
  const dim3 grid(p.blocks, p.slices);
  if (backward) wide_kernel<T, VE, K, true><<<grid, 256, 0, st>>>(a);
  else wide_kernel<T, VE, K, false><<<grid, 256, 0, st>>>(a);
}
template <typename T, int VE>
void launch_wide(const Args& a, const Plan& p, bool backward, hipStream_t st) {
  if (p.per_thread == 1) launch_wide<T, VE, 1>(a, p, backward, st);
  else if (p.per_thread == 2) launch_wide<T, VE, 2>(a, p, backward, st);
  else launch_wide<T, VE, 4>(a, p, backward, st);
}

template <typename T, int VE>
void launch_long(const Args& a, const Plan& p, bool backward, hipStream_t st) {
  const unsigned grid = (unsigned)((long long)a.batch * p.blocks * p.slices), pairs = (unsigned)(((long long)a.batch * a.groups + 3) / 4);
  const unsigned join = pairs < LAUNCH ? pairs : LAUNCH;
  if (backward) {
    if (p.records < a.batch) long_sum_kernel<T, VE, true><<<(unsigned)((long long)p.records * p.slices), 256, 0, st>>>(a, p);
    else long_sum_kernel<T, VE, false><<<grid, 256, 0, st>>>(a, p);
    if (a.dx == nullptr) return;
    long_join_kernel<true><<<join, 256, 0, st>>>(a, p);
    long_dx_kernel<T, VE><<<grid, 256, 0, st>>>(a, p);
  } else {
    long_stat_kernel<T, VE><<<grid, 256, 0, st>>>(a, p);
    long_join_kernel<false><<<join, 256, 0, st>>>(a, p);
    long_apply_kernel<T, VE><<<grid, 256, 0, st>>>(a, p);
  }
}

template <typename T>
void launch(const Args& a, const Plan& p, bool backward, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  if (p.form == ROWS) {
    if (p.pow2) launch_rows<T, N, true>(a, p, backward, st);
    else if (p.ve > 1) launch_rows<T, N, false>(a, p, backward, st);
    else launch_rows<T, 1, false>(a, p, backward, st);
  } else if (p.form == WIDE) {
    if (p.ve == 1) launch_wide<T, 1>(a, p, backward, st);
    else launch_wide<T, N>(a, p, backward, st);
  } else if (p.form == SLAB) {
    const int most = backward && p.records < a.batch ? a.batch : (int)LAUNCH / p.slices > 1 ? (int)LAUNCH / p.slices : 1;
    for (int first = 0; first < a.batch; first += most) {
      const Args part = samples<T>(a, first, a.batch - first < most ? a.batch - first : most);
      if (p.ve == 1) launch_slab<T, 1>(part, p, backward, st);
      else launch_slab<T, N>(part, p, backward, st);
      if (a.batch - first <= most) break;
    }
  } else {
    if (p.ve == 1) launch_long<T, 1>(a, p, backward, st);
    else launch_long<T, N>(a, p, backward, st);
  }
  if (backward && a.dweight != nullptr) {
    const float* records = a.work + work_floats(a, p, false);
    param_grad_kernel<T><<<(2 * a.channels + 15) / 16, 1024, 0, st>>>(a, records, p.records);
  }
}

int run(const Args* args, bool backward, const char* entry, void* stream) {
  if (args == nullptr || !sizes_ok(*args)) return fail(entry, -22);
  const Args& a = *args;
  if (a.x == nullptr || a.stats == nullptr || (reinterpret_cast<uintptr_t>(a.stats) | reinterpret_cast<uintptr_t>(a.work)) % 8 != 0 || a.activation < 0 || a.activation > 3 || (a.weight == nullptr) != (a.bias == nullptr) ||
      (a.weight_type != TYPE_F32 && a.weight_type != a.type) || !(a.eps >= 0.0f))
    return fail(entry, -22);
  if (!backward && a.y == nullptr) return fail(entry, -22);
  if (backward && (a.dy == nullptr || (a.dx == nullptr && a.dweight == nullptr) || (a.dweight == nullptr) != (a.dbias == nullptr) ||
                   (a.dweight != nullptr && a.weight == nullptr))) return fail(entry, -22);
  const Plan p = plan(a);
  const uintptr_t own = backward ? reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.dx) : reinterpret_cast<uintptr_t>(a.y);
  if (p.ve > 1 && own % 16 != 0) return fail(entry, -22);
  if (a.work == nullptr && work_floats(a, p, backward && a.dweight != nullptr) > 0) return fail(entry, -22);
  // workgroups of one launch (rows and wide: at most a few thousand; slab: several launches)
  if (p.form == LONG && (long long)a.batch * p.slices * p.blocks > 2LL * LAUNCH - 1) return fail(entry, -22);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.type == TYPE_F32) launch<float>(a, p, backward, st);
  else if (a.type == TYPE_BF16) launch<__bf16>(a, p, backward, st);
  else launch<_Float16>(a, p, backward, st);
  return launch_status(entry);
}

}  // namespace gn
}  // namespace is

extern "C" {

long long is_group_norm_work_floats(const IsGroupNorm* args, int backward) {
  if (args == nullptr || !is::gn::sizes_ok(*args)) return 0;
  return is::gn::work_floats(*args, is::gn::plan(*args), backward != 0);
}
int is_group_norm_fwd(const IsGroupNorm* args, void* stream) { return is::gn::run(args, false, "is_group_norm_fwd", stream); }
int is_group_norm_bwd(const IsGroupNorm* args, void* stream) { return is::gn::run(args, true, "is_group_norm_bwd", stream); }

}  // extern "C"
