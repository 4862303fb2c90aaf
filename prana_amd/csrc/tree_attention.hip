// Attention of drafted tokens over the caches of several sequences
// (prana_attention_tree). Drafted token i of a sequence with n rows in its
// cache sees row t when t < n or bit t - n of its mask word is set.
// One wave per drafted token and head.
#include <algorithm>

#include "common.h"
#include "serving.h"

namespace prana {

namespace {

constexpr int kTrSeqs = 64;

struct TreeSeq {
  const void *k, *v;
  const float *ks, *vs;
  uint32_t past, tok0, tokens;
};

struct TreeArgs {
  const float* q;
  const uint64_t* mask;
  float* out;
  uint32_t n_heads, n_kv, group, hd;
  float scale;
  TreeSeq seq[kTrSeqs];
};

template <bool Q8>
__global__ __launch_bounds__(64) void tree_kernel(TreeArgs a) {
  const TreeSeq& sq = a.seq[blockIdx.z];
  const uint32_t i = blockIdx.x, lane = threadIdx.x;
  if (i >= sq.tokens) return;
  const uint32_t head = blockIdx.y, kvh = head / a.group;
  const bool live = lane * 4 < a.hd;
  const size_t at = ((static_cast<size_t>(sq.tok0) + i) * a.n_heads + head) * a.hd + lane * 4;
  const uint64_t own = sq.tokens == 64 ? ~0ull : (1ull << sq.tokens) - 1;
  const uint64_t bits = (a.mask ? a.mask[sq.tok0 + i] : (2ull << i) - 1) & own;
  float q[4] = {}, acc[4] = {}, m = -INFINITY, l = 0.0f;
  if (live)
    for (int j = 0; j < 4; j++) q[j] = a.q[at + j];
  for (uint32_t t = 0; t < sq.past + sq.tokens; t++) {
    if (t >= sq.past && !((bits >> (t - sq.past)) & 1)) continue;
    const size_t row = static_cast<size_t>(t) * a.n_kv + kvh, kt = row * a.hd + lane * 4;
    float s = 0.0f, v[4] = {};
    if (live)
      for (int j = 0; j < 4; j++) {
        if constexpr (Q8) {
          s = fmaf(q[j], static_cast<float>(static_cast<const int8_t*>(sq.k)[kt + j]), s);
          v[j] = static_cast<float>(static_cast<const int8_t*>(sq.v)[kt + j]) * sq.vs[row];
        } else {
          s = fmaf(q[j], f16_operand(static_cast<const uint16_t*>(sq.k)[kt + j]), s);
          v[j] = f16_operand(static_cast<const uint16_t*>(sq.v)[kt + j]);
        }
      }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    s *= a.scale;
    if constexpr (Q8) s *= sq.ks[row];
    const float mn = fmaxf(m, s), al = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
    l = fmaf(l, al, p);
    for (int j = 0; j < 4; j++) acc[j] = fmaf(acc[j], al, p * v[j]);
    m = mn;
  }
  if (live)
    for (int j = 0; j < 4; j++) a.out[at + j] = l == 0.0f ? 0.0f : acc[j] / l;
}

}  // namespace

size_t attention_tree_floats(const size_t*, const size_t*, size_t, size_t, size_t, size_t) { return 0; }

int launch_attention_tree(const float* q, bool q8, const prana_kv* kv, const size_t* past, const size_t* n_tree,
                          size_t n_seq, const uint64_t* mask, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                          float* out, float*, hipStream_t s) {
  TreeArgs a{q, mask, out, static_cast<uint32_t>(n_heads), static_cast<uint32_t>(n_kv_heads),
             static_cast<uint32_t>(n_heads / n_kv_heads), static_cast<uint32_t>(head_dim),
             1.0f / sqrtf(static_cast<float>(head_dim))};
  size_t tok = 0, n = 0;
  uint32_t most = 0;
  for (size_t i = 0; i <= n_seq; i++) {
    if (i == n_seq || n == kTrSeqs) {
      if (n) {
        const dim3 grid(most, static_cast<uint32_t>(n_heads), static_cast<uint32_t>(n));
        if (q8)
          hipLaunchKernelGGL(tree_kernel<true>, grid, dim3(64), 0, s, a);
        else
          hipLaunchKernelGGL(tree_kernel<false>, grid, dim3(64), 0, s, a);
        PRANA_LAUNCH_CHECK();
      }
      n = 0;
      most = 0;
      if (i == n_seq) break;
    }
    if (!n_tree[i]) continue;
    a.seq[n++] = TreeSeq{kv[i].k, kv[i].v, kv[i].k_scales, kv[i].v_scales, static_cast<uint32_t>(past[i]),
                         static_cast<uint32_t>(tok), static_cast<uint32_t>(n_tree[i])};
    most = std::max(most, static_cast<uint32_t>(n_tree[i]));
    tok += n_tree[i];
  }
  return kOk;
}

}  // namespace prana
