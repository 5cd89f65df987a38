// Rotary positions: pairs of a head's elements turned by position * frequency.
//
//   (a, b) -> amplitude (a cos t - b sin t, a sin t + b cos t),  t = position * freq[p]
//
// The angle of a far position needs more than 32 bits (position 1e6 at frequency 1 leaves 0.06 radians of error in fp32): it is formed in
// turns in 64 bits, reduced to half a turn either side, and only then taken to 32 bits for sin / cos.  One sin / cos per token and pair, kept in
// LDS and shared by all heads of q and k; beyond that the kernel moves bytes: every element read once and written once, 16 bytes per access.
// Measured: (4, 8192, 32 + 8 heads of 128, bf16) 152 us each way = 4.4 TB/s (a copy: 5.1); (128, 283, 2 + 2 heads of 32, fp32) 12.4 us; single tokens
// 3.9 us, a launch.
#include "../../include/immunostruct_hip.h"
#include "tiles16.h"

namespace is {

constexpr int ROT_PAIRS = 256;      // pairs of the widest turned part
struct RotaryArgs {
  const void *x[2];
  void* out[2];
  long long s_b[2], s_n[2], s_h[2];
  const void* positions;
  long long pos_b, pos_n;
  int heads[2];
  int batch, n, width, part, positions64, tokens;      // tokens: of one workgroup
  float amplitude, sign;
  double turns[ROT_PAIRS];      // frequencies in turns a position
};

// VEC: everything is a multiple of 16 bytes (pointers, strides, width, part and, for half pairs, part / 2)
template <typename T, bool HALF, bool VEC>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  constexpr int N = VEC ? Vec<T>::N : 1;
  extern __shared__ float2 turn[];      // [token][pair]: amplitude * (cos, sin)
  const int pairs = a.part / 2, tid = threadIdx.x;
  const long long token0 = (long long)blockIdx.x * a.tokens, total = (long long)a.batch * a.n;
  const int count = (int)(total - token0 < a.tokens ? total - token0 : a.tokens);
  for (int i = tid; i < count * pairs; i += 256) {
    const int tk = i / pairs, p = i - tk * pairs;
    const long long token = token0 + tk, b = token / a.n, row = token - b * a.n;
    long long pos = row;
    if (a.positions != nullptr) {
      const long long at = b * a.pos_b + row * a.pos_n;
      pos = a.positions64 ? reinterpret_cast<const long long*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
    }
    double t = (double)pos * a.turns[p];
    t -= rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    turn[i] = make_float2(c * a.amplitude, s * a.sign * a.amplitude);
  }
  __syncthreads();
  // items of a head: pairs of chunks (half) or chunks of pairs (interleaved; scalar: single pairs), then chunks to copy
  const int turned = HALF || !VEC ? pairs / N : a.part / N, items = turned + (a.width - a.part) / N;
  const int all_heads = a.heads[0] + a.heads[1];
  const int work = count * all_heads * items;
  for (int i = tid; i < work; i += 256) {
    const int th = i / items, item = i - th * items, tk = th / all_heads, h0 = th - tk * all_heads;
    const int w = h0 >= a.heads[0] ? 1 : 0, h = h0 - (w ? a.heads[0] : 0);
    const long long token = token0 + tk, b = token / a.n, row = token - b * a.n;
    const T* x = reinterpret_cast<const T*>(a.x[w]) + b * a.s_b[w] + row * a.s_n[w] + h * a.s_h[w];
    T* y = reinterpret_cast<T*>(a.out[w]) + (token * a.heads[w] + h) * a.width;
    const float2* cs = turn + tk * pairs;
    if (item >= turned) {
      const int at = a.part + (item - turned) * N;
      if constexpr (VEC) *reinterpret_cast<u32x4_t*>(y + at) = *reinterpret_cast<const u32x4_t*>(x + at);
      else y[at] = x[at];
    } else if constexpr (VEC) {
      float u[N], v[N];
      if constexpr (HALF) {
        const int p = item * N;
        Vec<T>::unpack(*reinterpret_cast<const u32x4_t*>(x + p), u);
        Vec<T>::unpack(*reinterpret_cast<const u32x4_t*>(x + p + pairs), v);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 q = cs[p + e];
          const float s = u[e] * q.x - v[e] * q.y;
          v[e] = u[e] * q.y + v[e] * q.x;
          u[e] = s;
        }
        *reinterpret_cast<u32x4_t*>(y + p) = Vec<T>::pack(u);
        *reinterpret_cast<u32x4_t*>(y + p + pairs) = Vec<T>::pack(v);
      } else {
        const int at = item * N;
        Vec<T>::unpack(*reinterpret_cast<const u32x4_t*>(x + at), u);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 q = cs[(at + e) >> 1];
          const float s = u[e] * q.x - u[e + 1] * q.y;
          u[e + 1] = u[e] * q.y + u[e + 1] * q.x;
          u[e] = s;
        }
        *reinterpret_cast<u32x4_t*>(y + at) = Vec<T>::pack(u);
      }
    } else {
      const int p0 = HALF ? item : 2 * item, p1 = HALF ? item + pairs : 2 * item + 1;
      const float2 q = cs[item];
      const float u = (float)x[p0], v = (float)x[p1];
      y[p0] = (T)(u * q.x - v * q.y);
      y[p1] = (T)(u * q.y + v * q.x);
    }
  }
}

template <typename T>
void launch_rotary(const RotaryArgs& a, bool half, bool vec, hipStream_t st) {
  const unsigned grid = (unsigned)(((long long)a.batch * a.n + a.tokens - 1) / a.tokens);
  const size_t lds = (size_t)a.tokens * (a.part / 2) * sizeof(float2);
  if (half) {
    if (vec) rotary_kernel<T, true, true><<<grid, 256, lds, st>>>(a);
    else rotary_kernel<T, true, false><<<grid, 256, lds, st>>>(a);
  } else {
    if (vec) rotary_kernel<T, false, true><<<grid, 256, lds, st>>>(a);
    else rotary_kernel<T, false, false><<<grid, 256, lds, st>>>(a);
  }
}

}  // namespace is

extern "C" int is_rotary(const void* q, long long q_b, long long q_n, long long q_h, void* q_out, int heads,
                         const void* k, long long k_b, long long k_n, long long k_h, void* k_out, int kv_heads,
                         const void* positions, int positions64, long long pos_b, long long pos_n, const double* freq,
                         int batch, int n, int width, int part, int interleaved, int inverse, float amplitude, int type, void* stream) {
  using namespace is;
  if (q == nullptr || q_out == nullptr || freq == nullptr || batch < 1 || n < 1 || heads < 1 || kv_heads < 0 || width < 1 || part < 2 ||
      part % 2 != 0 || part > width || part / 2 > ROT_PAIRS || width > 65536 || heads > 65536 || kv_heads > 65536 || type < TYPE_F32 || type > TYPE_F16 ||
      (kv_heads > 0 && (k == nullptr || k_out == nullptr)))
    return fail("is_rotary", -22);
  RotaryArgs a;
  a.x[0] = q, a.x[1] = k, a.out[0] = q_out, a.out[1] = k_out;
  a.s_b[0] = q_b, a.s_n[0] = q_n, a.s_h[0] = q_h, a.s_b[1] = k_b, a.s_n[1] = k_n, a.s_h[1] = k_h;
  a.heads[0] = heads, a.heads[1] = kv_heads;
  a.positions = positions, a.positions64 = positions64, a.pos_b = pos_b, a.pos_n = pos_n;
  a.batch = batch, a.n = n, a.width = width, a.part = part;
  a.amplitude = amplitude, a.sign = inverse ? -1.0f : 1.0f;
  for (int p = 0; p < part / 2; ++p) a.turns[p] = freq[p] / 6.283185307179586476925286766559;
  // tokens of a workgroup: about 4 items of 16 bytes a thread, sin / cos in at most 16 KB of LDS
  const long long bytes = (long long)(heads + kv_heads) * width * (type == TYPE_F32 ? 4 : 2);
  long long tokens = 16384 / bytes;
  const long long most = 16384 / (part / 2 * (long long)sizeof(float2));
  tokens = tokens < 1 ? 1 : tokens;
  tokens = tokens > most ? most : tokens;
  a.tokens = (int)tokens;
  const long long total = (long long)batch * n;
  if ((total + tokens - 1) / tokens > 0xffffffLL || (heads + kv_heads) * (long long)width * tokens > 0x7fffffffLL) return fail("is_rotary", -22);
  const int N = type == TYPE_F32 ? 4 : 8;
  const long long strides = q_b | q_n | q_h | (kv_heads > 0 ? k_b | k_n | k_h : 0);
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) |
                         (kv_heads > 0 ? reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) : 0);
  const bool vec = strides % N == 0 && ptrs % 16 == 0 && width % N == 0 && (interleaved ? part : part / 2) % N == 0 && part % N == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (type == TYPE_F32) launch_rotary<float>(a, !interleaved, vec, st);
  else if (type == TYPE_BF16) launch_rotary<__bf16>(a, !interleaved, vec, st);
  else launch_rotary<_Float16>(a, !interleaved, vec, st);
  return launch_status("is_rotary");
}
