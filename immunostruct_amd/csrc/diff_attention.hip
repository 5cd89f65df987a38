// Differential attention: the C ABI's entry points (kernels and their reasons: diff_attention.h).
#include "diff_attention.h"

using namespace is;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// what both directions check; fills in the derived fields
int prepare(da::Args& a) {
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.lam == nullptr) return -22;
  if (a.batch < 1 || a.nq < 1 || a.nk < 1 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.d < 1 || a.dv < 1) return -22;
  if (a.type < TYPE_F32 || a.type > TYPE_F16 || (a.lam_type != TYPE_F32 && a.lam_type != a.type) || a.causal < 0 || a.causal > 2) return -22;
  if (!(a.scale > 0.0f) || !(a.scale < 2e38f) || a.splits < 1 || a.splits > 64 || a.row_splits < 1) return -22;
  a.group = a.heads / a.kv_heads;
  a.group_magic = 0xffffffffu / (unsigned)a.group;
  const long long rows = (long long)a.nq * a.group, big = 0x7fffff00LL;
  const int n = a.type == TYPE_F32 ? 4 : 8, size = 16 / n;
  // a launch has to stay below 2^32 threads: 128 for 32 rows or keys, up to 256 for a row that is joined, one for an element of joined key gradients
  const long long tiles = 0x1ffffffLL;
  if (rows > big || a.nk > big || (rows / 32 + 4) * a.splits * a.kv_heads > tiles / a.batch || (rows + 3) * a.kv_heads > big / a.batch ||
      (a.nk / 32 + 4LL) * a.row_splits * a.kv_heads > tiles / a.batch || (a.splits > 1 && (rows + 3) * a.kv_heads > tiles / 2 / a.batch) ||
      (a.row_splits > 1 && (a.nk * (2LL * a.d + a.dv) + 255) / 256 * a.kv_heads > tiles / 2 / a.batch)) return -22;
  a.rows = (int)rows;
  // a tile's rows lie within 31 bits of its first
  const long long near = 0x7fffffffLL / size;
  if (a.q_n < 0 || a.q_h < 0 || a.k_n < 0 || a.k_h < 0 || a.v_n < 0 || a.k_h > near / 4 || a.q_n > near / 64 || a.k_n > near / 64 || a.v_n > near / 64 ||
      a.q_h > near / 4 / a.group || (long long)a.heads * a.dv > near / 64) return -22;
  const long long strides = a.q_b | a.q_n | a.q_h | a.k_b | a.k_n | a.k_h | a.v_b | a.v_n | a.v_h;
  a.vec = aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.o) && aligned16(a.maps) && aligned16(a.d_o) && aligned16(a.dq) &&
          aligned16(a.dk) && aligned16(a.dv_out) && strides % n == 0 && a.d % n == 0 && a.dv % n == 0;
  return da::class_of(a) == 0 ? -38 : 0;
}

int run(const da::Args& a, bool backward, const char* entry, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.type == TYPE_F32) da::run_f32(a, backward, st);
  else if (a.type == TYPE_BF16) da::run_bf16(a, backward, st);
  else da::run_f16(a, backward, st);
  return launch_status(entry);
}

}  // namespace

extern "C" {

// Splits of the keys, where the rows alone do not fill the chip.  Up to 32 rows (single tokens) a workgroup is one pair of waves and the call is
// bound by the cache's bytes: 1024 workgroups, at least 128 keys each.  More rows: 256 times 128 rows in all (the kernels take them as two workgroups of 64),
// and only while a split has work enough to pay for leaving its sums in memory: 512 keys in the 16-bit types, 128 in the 8 to 16 times slower 32-bit one.
// Measured (us) for at least 128 / 512 / 1024 keys: (1, 512 over 4096, 8 / 2 heads, 64) bf16 61 / 61 / 55, (2, 300 over 300, 8, 64) bf16 30 / 16 / 16, (1, 128
// over 2048, 4 / 1, 64) bf16 24 / 26 / 38, (1, 2048 over 2048, 2, 64) fp32 67 / 75 / 123; with twice the splits the last takes 94.
int is_diff_attention_splits(int batch, int kv_heads, int rows, int nk, int type) {
  if (batch < 1 || kv_heads < 1 || rows < 1 || nk < 1) return 1;
  const long long groups = (rows <= 32 ? 1LL : (rows + 127LL) / 128) * kv_heads * batch;
  const long long want = rows <= 32 ? 1024 / groups : groups < 128 ? 256 / groups : 1, least = rows <= 32 || type == TYPE_F32 ? 128 : 512;
  const long long most = (nk + least - 1) / least, s = want < most ? want : most;
  return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}

// Row splits of the key gradients, counted in tiles of 128 keys, which the kernels take as one workgroup (16-bit heads of 33 ... 64) or two (others).  With a
// mask the first tiles have all the work, two parts of each fill the gaps the last ones leave; few key tiles are split until 256 are there, at least
// 256 rows each, 16 parts at most.  Counted in the workgroups launched instead, the key gradients (with the row sums, us) went 219 -> 196 at (5, 517 over 1531,
// 6 / 2 heads, 128) fp16 and 210 -> 200 at (1, 2048, 8 / 2, 128) bf16, no mask, but 90 -> 105 at (2, 1024, 8 / 2, 128) bf16, 62 -> 73 at (1, 1500, 4 / 1, 128)
// fp16 and 88 -> 121 at (1, 2048, 2, 64) fp32, causal.
int is_diff_attention_row_splits(int batch, int kv_heads, int rows, int nk, int causal) {
  if (batch < 1 || kv_heads < 1 || rows < 1 || nk < 1) return 1;
  const long long groups = (nk + 127LL) / 128 * kv_heads * batch, most = (rows + 255LL) / 256;
  long long s = groups <= 128 ? 256 / groups : causal != 0 && groups < 1024 ? 2 : 1;
  s = s < most ? s : most;
  return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

long long is_diff_attention_row_work_floats(int batch, int kv_heads, int nk, int d, int dv, int row_splits) {
  return row_splits <= 1 ? 0 : (long long)row_splits * batch * kv_heads * nk * (2 * d + dv);
}

long long is_diff_attention_work_floats(int batch, int kv_heads, int rows, int dv, int splits) {
  return splits <= 1 ? 0 : 2LL * batch * kv_heads * splits * rows * (dv + 2);
}

int is_diff_attention_fwd(const IsDiffAttention* args, void* stream) {
  if (args == nullptr) return fail("is_diff_attention_fwd", -22);
  da::Args a = *args;
  a.d_o = nullptr;
  a.dq = a.dk = a.dv_out = a.dlam = nullptr;
  a.row_splits = 1;
  const int rc = prepare(a);
  if (rc != 0) return fail("is_diff_attention_fwd", rc);
  if (a.o == nullptr || (a.lse == nullptr) != (a.maps == nullptr) || (a.splits > 1 && a.work == nullptr)) return fail("is_diff_attention_fwd", -22);
  return run(a, false, "is_diff_attention_fwd", stream);
}

int is_diff_attention_bwd(const IsDiffAttention* args, void* stream) {
  if (args == nullptr) return fail("is_diff_attention_bwd", -22);
  da::Args a = *args;
  a.splits = 1;
  a.o = nullptr;
  const int rc = prepare(a);
  if (rc != 0) return fail("is_diff_attention_bwd", rc);
  if (a.maps == nullptr || a.lse == nullptr || a.d_o == nullptr || a.dots == nullptr || (a.dk == nullptr) != (a.dv_out == nullptr) ||
      (a.dq == nullptr && (a.dk == nullptr || a.dlam != nullptr)) || (a.dk != nullptr && a.row_splits > 1 && a.work == nullptr))
    return fail("is_diff_attention_bwd", -22);
  return run(a, true, "is_diff_attention_bwd", stream);
}

}  // extern "C"
