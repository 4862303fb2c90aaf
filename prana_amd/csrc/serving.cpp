// Argument checks of the serving entry points: host code without device calls,
// so that a call is refused before anything is launched, with or without a GPU.
#include "serving.h"

#include <string>

#include "common.h"

namespace prana {

namespace {

constexpr size_t kMaxRows = size_t{1} << 30;  // rows (times heads) of one sequence: indices and grids fit 32 bits

constexpr size_t kMaxStride = size_t{1} << 24;  // row strides: 63 rows' bytes fit 32 bits

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int refuse(const char* what, const std::string& why) { return fail(kErrInvalid, std::string(what) + ": " + why); }

}  // namespace

int check_heads(const char* what, size_t n_heads, size_t n_kv_heads, size_t head_dim) {
  if (n_kv_heads == 0 || n_heads == 0 || n_heads % n_kv_heads != 0)
    return refuse(what, "n_heads must be a positive multiple of n_kv_heads");
  if (head_dim == 0 || head_dim > 256 || head_dim % 8 != 0)
    return refuse(what, "head_dim must be a multiple of 8 up to 256");
  if (n_heads > 65535) return refuse(what, "more than 65535 heads");
  return kOk;
}

int check_attention_packed(const void* q, const uint16_t* k, const uint16_t* v, int type, const size_t* seq_lens,
                           size_t n_seq, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t ld_q,
                           size_t ld_kv, size_t ld_out, const void* out) {
  const char* what = "attention_packed";
  if (type != PRANA_F32 && type != PRANA_F16) return refuse(what, "type must be PRANA_F32 or PRANA_F16");
  if (int rc = check_heads(what, n_heads, n_kv_heads, head_dim)) return rc;
  if (n_seq && !seq_lens) return refuse(what, "null seq_lens");
  size_t total = 0;
  for (size_t i = 0; i < n_seq; i++) {
    if (seq_lens[i] > kMaxRows || seq_lens[i] * n_heads > kMaxRows ||
        packed_lanes(seq_lens[i], n_heads, n_kv_heads, head_dim) > 0xffffffffu)
      return refuse(what, "sequence " + std::to_string(i) + " is too long");
    total += seq_lens[i];
    if (total > 0xffffffffu) return refuse(what, "more than 2^32 - 1 rows");
  }
  if (total == 0) return kOk;
  if (!q || !k || !v || !out) return refuse(what, "null buffer");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
    return refuse(what, "buffers must be 16-byte aligned");
  const size_t per16 = type == PRANA_F32 ? 4 : 8;
  if (ld_q % per16 || ld_out % per16 || ld_kv % 8) return refuse(what, "row strides must be multiples of 16 bytes");
  if (ld_q < n_heads * head_dim || ld_out < n_heads * head_dim || ld_kv < n_kv_heads * head_dim)
    return refuse(what, "a row stride is shorter than its row");
  if (ld_q > kMaxStride || ld_out > kMaxStride || ld_kv > kMaxStride) return refuse(what, "a row stride is too long");
  return kOk;
}

int check_kv_q8(const char* what, const prana_kv* kv, const size_t* first_rows, const size_t* n_rows, size_t n_seq,
                size_t n_kv_heads, size_t head_dim, const void* k, const void* v, size_t ld, size_t size) {
  if (int rc = check_heads(what, n_kv_heads, n_kv_heads, head_dim)) return rc;
  if (n_seq && (!kv || !first_rows || !n_rows)) return refuse(what, "null argument");
  size_t total = 0;
  for (size_t i = 0; i < n_seq; i++) {
    if (n_rows[i] == 0) continue;
    const std::string seq = "sequence " + std::to_string(i);
    if (kv[i].rows > kMaxRows) return refuse(what, seq + ": cache of more than 2^30 rows");
    if (n_rows[i] > kv[i].rows || first_rows[i] > kv[i].rows - n_rows[i])
      return refuse(what, seq + ": rows past the end of the cache");
    if (!kv[i].k || !kv[i].v || !kv[i].k_scales || !kv[i].v_scales) return refuse(what, seq + ": null cache pointer");
    if (!aligned(kv[i].k, 16) || !aligned(kv[i].v, 16)) return refuse(what, seq + ": caches must be 16-byte aligned");
    if (!aligned(kv[i].k_scales, 4) || !aligned(kv[i].v_scales, 4))
      return refuse(what, seq + ": scales must be 4-byte aligned");
    total += n_rows[i];
    if (total > 0xffffffffu) return refuse(what, "more than 2^32 - 1 rows");
  }
  if (total == 0) return kOk;
  if (!k || !v) return refuse(what, "null buffer");
  if (!aligned(k, 16) || !aligned(v, 16)) return refuse(what, "buffers must be 16-byte aligned");
  if (ld > kMaxStride) return refuse(what, "row stride too long");
  if (ld * size % 16) return refuse(what, "row stride must be a multiple of 16 bytes");
  if (ld < n_kv_heads * head_dim) return refuse(what, "row stride shorter than a row");
  return kOk;
}

int check_tree_sizes(const size_t* past, const size_t* n_tree, size_t n_seq, size_t n_heads, size_t n_kv_heads,
                     size_t head_dim) {
  const char* what = "attention_tree";
  if (int rc = check_heads(what, n_heads, n_kv_heads, head_dim)) return rc;
  if (n_seq && (!past || !n_tree)) return refuse(what, "null sizes");
  size_t total = 0;
  for (size_t i = 0; i < n_seq; i++) {
    const std::string seq = "sequence " + std::to_string(i);
    if (n_tree[i] > kMaxTree) return refuse(what, seq + ": more than 64 drafted tokens");
    if (past[i] > kMaxRows - kMaxTree) return refuse(what, seq + " is too long");
    total += n_tree[i];
    if (total * n_heads > kMaxRows) return refuse(what, "too many drafted tokens");
  }
  return kOk;
}

int check_attention_tree(const float* q, int kv_type, const prana_kv* kv, const size_t* past, const size_t* n_tree,
                         size_t n_seq, const uint64_t* mask, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                         const float* out, const void* workspace, size_t workspace_bytes) {
  const char* what = "attention_tree";
  if (kv_type != PRANA_KV_F16 && kv_type != PRANA_KV_Q8)
    return refuse(what, "kv_type must be PRANA_KV_F16 or PRANA_KV_Q8");
  if (int rc = check_tree_sizes(past, n_tree, n_seq, n_heads, n_kv_heads, head_dim)) return rc;
  if (n_seq && !kv) return refuse(what, "null caches");
  bool any = false;
  for (size_t i = 0; i < n_seq; i++) {
    if (n_tree[i] == 0) continue;
    any = true;
    const std::string seq = "sequence " + std::to_string(i);
    if (kv[i].rows > kMaxRows) return refuse(what, seq + ": cache of more than 2^30 rows");
    if (n_tree[i] > kv[i].rows || past[i] > kv[i].rows - n_tree[i])
      return refuse(what, seq + ": rows past the end of the cache");
    if (!kv[i].k || !kv[i].v) return refuse(what, seq + ": null cache pointer");
    if (!aligned(kv[i].k, 16) || !aligned(kv[i].v, 16)) return refuse(what, seq + ": caches must be 16-byte aligned");
    if (kv_type == PRANA_KV_Q8) {
      if (!kv[i].k_scales || !kv[i].v_scales) return refuse(what, seq + ": null scales");
      if (!aligned(kv[i].k_scales, 4) || !aligned(kv[i].v_scales, 4))
        return refuse(what, seq + ": scales must be 4-byte aligned");
    }
  }
  if (!any) return kOk;
  if (!q || !out) return refuse(what, "null buffer");
  if (!aligned(q, 16) || !aligned(out, 16)) return refuse(what, "q and out must be 16-byte aligned");
  if (!aligned(mask, 8)) return refuse(what, "mask must be 8-byte aligned");
  const size_t need = attention_tree_floats(past, n_tree, n_seq, n_heads, n_kv_heads, head_dim) * sizeof(float);
  if (need > (size_t{1} << 42)) return refuse(what, "too many drafted tokens over too long caches");
  if (need && !workspace) return refuse(what, "null workspace");
  if (!aligned(workspace, 16)) return refuse(what, "workspace must be 16-byte aligned");
  if (workspace_bytes < need)
    return refuse(what, "workspace of " + std::to_string(workspace_bytes) + " bytes; " + std::to_string(need) +
                            " needed");
  return kOk;
}

}  // namespace prana
