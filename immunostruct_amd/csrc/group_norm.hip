// Group norm with an activation, channels last (batch, n, channels), statistics over a sample's valid rows and a group's channels.
//
//   xhat = (x - mean) rstd,  z = xhat w + b,  y = act(z)
//   dz = dy act'(z),  dw = sum dz xhat,  db = sum dz,  t = dz w,  dx = rstd (t - mean(t) - xhat mean(t xhat))
#include "../../include/immunostruct_hip.h"
#include "tiles16.h"

namespace is {
namespace gn {

typedef IsGroupNorm Args;

__device__ __forceinline__ int length_of(const Args& a, int b) {
  const int n = a.lengths != nullptr ? a.lengths[b] : a.n;
  return n < 0 ? 0 : (n > a.n ? a.n : n);
}
__device__ __forceinline__ float param(const void* p, int type, int c, float other) {
  if (p == nullptr) return other;
  if (type == TYPE_F32) return reinterpret_cast<const float*>(p)[c];
  if (type == TYPE_BF16) return (float)reinterpret_cast<const __bf16*>(p)[c];
  return (float)reinterpret_cast<const _Float16*>(p)[c];
}
__device__ __forceinline__ void put(void* p, int type, int c, float v) {
  if (type == TYPE_F32) reinterpret_cast<float*>(p)[c] = v;
  else if (type == TYPE_BF16) reinterpret_cast<__bf16*>(p)[c] = (__bf16)v;
  else reinterpret_cast<_Float16*>(p)[c] = (_Float16)v;
}
__device__ __forceinline__ float act(float z, int kind) {
  if (kind == 1) return z / (1.0f + __expf(-z));
  if (kind == 2) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752440f));
  if (kind == 3) return z > 0.0f ? z : (z != z ? z : 0.0f);
  return z;
}
__device__ __forceinline__ float act_slope(float z, int kind) {
  if (kind == 1) {
    const float s = 1.0f / (1.0f + __expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  if (kind == 2) return 0.5f * (1.0f + erff(z * 0.70710678118654752440f)) + z * 0.39894228040143267794f * __expf(-0.5f * z * z);
  if (kind == 3) return z > 0.0f ? 1.0f : 0.0f;
  return 1.0f;
}
// sum over the 256 threads, in every thread
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = sum_over_r(v);
  v += other_half(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}

// one workgroup per (sample, group), any shape
template <typename T>
__global__ __launch_bounds__(256) void fwd_any_kernel(const Args a) {
  __shared__ float scratch[4];
  const int b = blockIdx.x / a.groups, g = blockIdx.x % a.groups, cg = a.channels / a.groups, len = length_of(a, b);
  const T* x = reinterpret_cast<const T*>(a.x) + b * a.x_b + g * cg;
  T* y = reinterpret_cast<T*>(a.y) + ((long long)b * a.n) * a.channels + g * cg;
  const long long count = (long long)len * cg, all = (long long)a.n * cg;
  float s = 0.0f;
  for (long long i = threadIdx.x; i < count; i += 256) s += (float)x[i / cg * a.x_n + i % cg];
  const float mean = block_sum(s, scratch) / (float)(count > 0 ? count : 1);
  s = 0.0f;
  for (long long i = threadIdx.x; i < count; i += 256) {
    const float d = (float)x[i / cg * a.x_n + i % cg] - mean;
    s += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum(s, scratch) / (float)(count > 0 ? count : 1) + a.eps);
  if (threadIdx.x == 0) {
    a.stats[2 * (long long)blockIdx.x] = mean;
    a.stats[2 * (long long)blockIdx.x + 1] = rstd;
  }
  for (long long i = threadIdx.x; i < all; i += 256) {
    const long long row = i / cg;
    const int c = (int)(i - row * cg);
    float v = 0.0f;
    if (row < len) {
      const float hat = ((float)x[row * a.x_n + c] - mean) * rstd;
      v = act(hat * param(a.weight, a.weight_type, g * cg + c, 1.0f) + param(a.bias, a.weight_type, g * cg + c, 0.0f), a.activation);
    }
    y[row * a.channels + c] = (T)v;
  }
}

// per (sample, group): the channels' sums of dz and dz xhat (part[sample][2][channels]), then dx
template <typename T>
__global__ __launch_bounds__(256) void bwd_any_kernel(const Args a, float* part) {
  __shared__ float scratch[4], col[2][256];
  const int b = blockIdx.x / a.groups, g = blockIdx.x % a.groups, cg = a.channels / a.groups, len = length_of(a, b);
  const T* x = reinterpret_cast<const T*>(a.x) + b * a.x_b + g * cg;
  const long long at = ((long long)b * a.n) * a.channels + g * cg;
  const T* dy = reinterpret_cast<const T*>(a.dy) + at;
  T* dx = reinterpret_cast<T*>(a.dx) + at;
  const float mean = a.stats[2 * (long long)blockIdx.x], rstd = a.stats[2 * (long long)blockIdx.x + 1];
  int lanes = 1;
  while (lanes < cg && lanes < 256) lanes *= 2;
  const int cl = threadIdx.x % lanes, rl = threadIdx.x / lanes, rows = 256 / lanes;
  float t1 = 0.0f, t2 = 0.0f;
  for (int c0 = 0; c0 < cg; c0 += lanes) {
    const int c = c0 + cl;
    const float w = c < cg ? param(a.weight, a.weight_type, g * cg + c, 1.0f) : 0.0f, bias = c < cg ? param(a.bias, a.weight_type, g * cg + c, 0.0f) : 0.0f;
    float s1 = 0.0f, s2 = 0.0f;
    if (c < cg)
      for (int row = rl; row < len; row += rows) {
        const float hat = ((float)x[row * a.x_n + c] - mean) * rstd;
        const float dz = (float)dy[row * (long long)a.channels + c] * act_slope(hat * w + bias, a.activation);
        s1 += dz;
        s2 += dz * hat;
      }
    t1 += s1 * w;
    t2 += s2 * w;
    __syncthreads();
    col[0][threadIdx.x] = s1;
    col[1][threadIdx.x] = s2;
    __syncthreads();
    if (part != nullptr && rl == 0 && c < cg) {
      for (int k = 1; k < rows; ++k) {
        s1 += col[0][k * lanes + cl];
        s2 += col[1][k * lanes + cl];
      }
      part[(2LL * b) * a.channels + g * cg + c] = s2;
      part[(2LL * b + 1) * a.channels + g * cg + c] = s1;
    }
  }
  const float count = (float)((long long)len * cg > 0 ? (long long)len * cg : 1);
  t1 = block_sum(t1, scratch) / count;
  t2 = block_sum(t2, scratch) / count;
  const long long all = (long long)a.n * cg;
  for (long long i = threadIdx.x; i < all; i += 256) {
    const long long row = i / cg;
    const int c = (int)(i - row * cg);
    float v = 0.0f;
    if (row < len) {
      const float w = param(a.weight, a.weight_type, g * cg + c, 1.0f);
      const float hat = ((float)x[row * a.x_n + c] - mean) * rstd;
      const float dz = (float)dy[row * a.channels + c] * act_slope(hat * w + param(a.bias, a.weight_type, g * cg + c, 0.0f), a.activation);
      v = rstd * (dz * w - t1 - hat * t2);
    }
    dx[row * a.channels + c] = (T)v;
  }
}

// dweight, dbias = the sums of `records` records [2][channels], in order
__global__ __launch_bounds__(256) void param_grad_kernel(const Args a, const float* part, int records) {
  __shared__ float sum[4][64];
  const int i = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6, total = 2 * a.channels;
  float s = 0.0f;
  if (i < total)
    for (int r = w; r < records; r += 4) s += part[(long long)r * total + i];
  sum[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && i < total) {
    const int l = threadIdx.x;
    s = (sum[0][l] + sum[1][l]) + (sum[2][l] + sum[3][l]);
    put(i < a.channels ? a.dweight : a.dbias, a.weight_type, i % a.channels, s);
  }
}

template <typename T>
void launch(const Args& a, bool backward, hipStream_t st) {
  const unsigned grid = (unsigned)((long long)a.batch * a.groups);
  if (!backward) {
    fwd_any_kernel<T><<<grid, 256, 0, st>>>(a);
    return;
  }
  bwd_any_kernel<T><<<grid, 256, 0, st>>>(a, a.weight != nullptr ? a.work : nullptr);
  if (a.weight != nullptr) param_grad_kernel<<<(2 * a.channels + 63) / 64, 256, 0, st>>>(a, a.work, a.batch);
}

bool sizes_ok(const Args& a) {
  return a.batch >= 1 && a.n >= 1 && a.channels >= 1 && a.groups >= 1 && a.channels % a.groups == 0 && a.channels <= (1 << 24) &&
         (long long)a.batch * a.groups <= 0x7fffffffLL && a.type >= TYPE_F32 && a.type <= TYPE_F16;
}

int run(const Args* args, bool backward, const char* entry, void* stream) {
  if (args == nullptr || !sizes_ok(*args)) return fail(entry, -22);
  const Args& a = *args;
  if (a.x == nullptr || a.stats == nullptr || a.activation < 0 || a.activation > 3 || (a.weight == nullptr) != (a.bias == nullptr) ||
      (a.weight_type != TYPE_F32 && a.weight_type != a.type) || !(a.eps >= 0.0f))
    return fail(entry, -22);
  if (!backward && a.y == nullptr) return fail(entry, -22);
  if (backward && (a.dy == nullptr || a.dx == nullptr || (a.weight != nullptr && (a.dweight == nullptr || a.dbias == nullptr)))) return fail(entry, -22);
  if (a.work == nullptr && is_group_norm_work_floats(args, backward ? 1 : 0) > 0) return fail(entry, -22);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.type == TYPE_F32) launch<float>(a, backward, st);
  else if (a.type == TYPE_BF16) launch<__bf16>(a, backward, st);
  else launch<_Float16>(a, backward, st);
  return launch_status(entry);
}

}  // namespace gn
}  // namespace is

extern "C" {

long long is_group_norm_work_floats(const IsGroupNorm* args, int backward) {
  if (args == nullptr || !is::gn::sizes_ok(*args)) return 0;
  return backward && args->weight != nullptr ? 2LL * args->batch * args->channels : 0;
}
int is_group_norm_fwd(const IsGroupNorm* args, void* stream) { return is::gn::run(args, false, "is_group_norm_fwd", stream); }
int is_group_norm_bwd(const IsGroupNorm* args, void* stream) { return is::gn::run(args, true, "is_group_norm_bwd", stream); }

}  // extern "C"
