// Causal attention of whole prompts packed behind one another
// (prana_attention_packed): per sequence and head
//   o_i = sum_{j <= i} p_ij v_j,  p_i = softmax_j(q_i . k_j / sqrt(hd)).
// One wave per query row and head: each lane holds 4 values of the head, the
// keys are visited in order with a running maximum and sum.
#include <algorithm>

#include "common.h"
#include "serving.h"

namespace prana {

namespace {

constexpr int kPkSeqs = 128;

struct PackedArgs {
  const void* q;
  const uint16_t *k, *v;
  void* out;
  size_t ld_q, ld_kv, ld_out;
  uint32_t n_seq, n_heads, group, hd;
  float scale;
  uint32_t start[kPkSeqs];
  uint32_t len[kPkSeqs];
  uint32_t block0[kPkSeqs];
};

template <bool HALF>
__global__ __launch_bounds__(256) void packed_kernel(PackedArgs a) {
  int lo = 0, hi = static_cast<int>(a.n_seq) - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.block0[mid] <= blockIdx.x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const uint32_t row = (blockIdx.x - a.block0[lo]) * 4 + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (row >= a.len[lo]) return;
  const uint32_t head = blockIdx.y, kvh = head / a.group;
  const bool live = lane * 4 < a.hd;
  float q[4] = {}, acc[4] = {};
  const size_t tok = static_cast<size_t>(a.start[lo]) + row;
  if (live)
    for (int j = 0; j < 4; j++) {
      const size_t at = tok * a.ld_q + head * a.hd + lane * 4 + j;
      q[j] = HALF ? f16_operand(static_cast<const uint16_t*>(a.q)[at]) : static_cast<const float*>(a.q)[at];
    }
  float m = -INFINITY, l = 0.0f;
  for (uint32_t t = 0; t <= row; t++) {
    const size_t at = (static_cast<size_t>(a.start[lo]) + t) * a.ld_kv + kvh * a.hd + lane * 4;
    float s = 0.0f;
    if (live)
      for (int j = 0; j < 4; j++) s = fmaf(q[j], f16_operand(a.k[at + j]), s);
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    s *= a.scale;
    const float mn = fmaxf(m, s), al = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
    l = fmaf(l, al, p);
    if (live)
      for (int j = 0; j < 4; j++) acc[j] = fmaf(acc[j], al, p * f16_operand(a.v[at + j]));
    m = mn;
  }
  if (live)
    for (int j = 0; j < 4; j++) {
      const size_t at = tok * a.ld_out + head * a.hd + lane * 4 + j;
      if (HALF)
        static_cast<uint16_t*>(a.out)[at] = f32_to_f16(acc[j] / l);
      else
        static_cast<float*>(a.out)[at] = acc[j] / l;
    }
}

}  // namespace

int launch_attention_packed(const void* q, const uint16_t* k, const uint16_t* v, bool half, const size_t* seq_lens,
                            size_t n_seq, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t ld_q,
                            size_t ld_kv, size_t ld_out, void* out, hipStream_t s) {
  PackedArgs a{q, k, v, out, ld_q, ld_kv, ld_out, 0, static_cast<uint32_t>(n_heads),
               static_cast<uint32_t>(n_heads / n_kv_heads), static_cast<uint32_t>(head_dim),
               1.0f / sqrtf(static_cast<float>(head_dim))};
  size_t at = 0, blocks = 0;
  for (size_t i = 0; i <= n_seq; i++) {
    if (i == n_seq || a.n_seq == kPkSeqs) {
      if (blocks) {
        const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(n_heads));
        if (half)
          hipLaunchKernelGGL(packed_kernel<true>, grid, dim3(256), 0, s, a);
        else
          hipLaunchKernelGGL(packed_kernel<false>, grid, dim3(256), 0, s, a);
        PRANA_LAUNCH_CHECK();
      }
      a.n_seq = 0;
      blocks = 0;
      if (i == n_seq) break;
    }
    if (seq_lens[i]) {
      a.start[a.n_seq] = static_cast<uint32_t>(at);
      a.len[a.n_seq] = static_cast<uint32_t>(seq_lens[i]);
      a.block0[a.n_seq++] = static_cast<uint32_t>(blocks);
      blocks += (seq_lens[i] + 3) / 4;
      at += seq_lens[i];
    }
  }
  return kOk;
}

}  // namespace prana
