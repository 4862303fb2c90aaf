// Causal attention of whole prompts packed behind one another
// (prana_attention_packed): per sequence and head
//   o_i = sum_{j <= i} p_ij v_j,  p_i = softmax_j(q_i . k_j / sqrt(w)).
//
// One pass over the keys with a running maximum and sum, on the f16 matrix
// cores. The rows of a sequence are its (token, query head of the group)
// pairs, so the heads that share a KV head share its tiles too; a workgroup
// takes 128 rows (32 per wave) and walks the keys up to its last token in
// tiles of kBN, staged through registers into LDS while the tile before is
// computed. Per tile and wave, with 32x32x16 products:
//   S^T = K Q^T : a lane holds one row's scores, 16 of each 32 keys, so the
//                 maximum and sum of a row are taken inside two lanes;
//   O^T += V^T P^T : the scores' registers are, as halves, the operand of
//                 this product (its keys in the order the registers hold
//                 them), and V comes out of LDS transposed to match. No
//                 probability moves between lanes.
// The maximum lags: it is raised, and the sums rescaled, only when a score
// passes it by more than 2^8, so probabilities are at most 256.
//
// f32 form: q * log2(e)/sqrt(w), normalised per row by a power of two, and the
// probabilities go in as two halves each (22 bits), twice the products.
#include <algorithm>
#include <cmath>
#include <vector>

#include "common.h"
#include "mfma_tile.h"
#include "seq_table.h"
#include "serving.h"

namespace prana {

namespace {

constexpr int kPkNT = 256;     // lanes of a workgroup
constexpr int kPkRows = 128;   // rows of a workgroup
constexpr float kLag = 8.0f;   // how far (log2) scores may pass the kept maximum
constexpr float kPShift = 7.0f;  // f32 form: probabilities are kept times 2^7 (at most 2^15), so that
                                 // the smaller half of one resolves 2^-32 of the largest

struct PackedArgs {
  const void* q;
  const uint16_t *k, *v;
  void* out;
  size_t ld_q, ld_kv, ld_out;
  uint32_t n_seq, n_kv, group, hd;
  float scale;  // log2(e) / sqrt(hd)
  uint32_t start[kTableSeqs];  // first packed row
  uint32_t len[kTableSeqs];
  uint32_t tile0[kTableSeqs];  // first row tile
};

// HDP: head width rounded up; the lanes past the real one hold zeros.
template <int HDP, int BN>
struct PkShape {
  static constexpr int kStepsQK = HDP / 16, kDimBlocks = HDP / 32, kKeyBlocks = BN / 32;
  static constexpr int kChunks = HDP / 8;  // 16-byte pieces of a row
  // K rows 16 bytes apart from a multiple of 32: the 16-byte reads of 8 rows
  // fall on different banks. V rows 64 bytes (mod 256) apart: so do the
  // 64-byte pieces of 4 rows that a transposing read takes.
  static constexpr int kLdK = HDP + 8;
  static constexpr int kLdV = HDP % 128 == 96 ? HDP : HDP + 32;
  static constexpr int kLoads = BN * kChunks / kPkNT;  // 16-byte pieces a lane stages of K (and of V)
};

template <int HDP, int BN, bool HALF>
__global__ __launch_bounds__(kPkNT, HDP <= 128 ? 2 : 1) void packed_kernel(PackedArgs a) {
  using S = PkShape<HDP, BN>;
  static_assert(BN * S::kChunks % kPkNT == 0, "a tile is a whole number of pieces per lane");
  __shared__ __attribute__((aligned(16))) uint16_t s_k[BN * S::kLdK];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[BN * S::kLdV];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  const uint32_t kvh = blockIdx.x % a.n_kv, tile = blockIdx.x / a.n_kv;
  const int sq = table_find(a.tile0, a.n_seq, tile);
  const uint32_t len = table_at(a.len, sq), rows = len * a.group;
  const uint32_t n_tiles = (rows + kPkRows - 1) / kPkRows;
  // the last tiles see the most keys: they go first
  const uint32_t row0 = (n_tiles - 1 - (tile - table_at(a.tile0, sq))) * kPkRows;
  const size_t base = table_at(a.start, sq);
  const uint32_t row_w = row0 + wave * 32;                       // the wave's first row
  const uint32_t row = min(row_w + n, rows - 1);                 // (rows past the end repeat the last one)
  const uint32_t tok = row / a.group, head = kvh * a.group + row % a.group;
  const uint32_t tok_first_wg = row0 / a.group;
  const uint32_t tok_last_wg = (min(row0 + kPkRows, rows) - 1) / a.group;
  const uint32_t tok_first = min(row_w, rows - 1) / a.group;      // of the wave
  const uint32_t tok_last = min(row_w + 31, rows - 1) / a.group;
  const uint32_t hd = a.hd;

  // Addresses: a uniform base per tile and a lane's 32-bit offset. Pieces past
  // the head's width repeat its last one (q is 0 there for K, and V columns
  // there are never stored).
  const uint16_t* kb = a.k + base * a.ld_kv + static_cast<size_t>(kvh) * hd;
  const uint16_t* vb = a.v + base * a.ld_kv + static_cast<size_t>(kvh) * hd;
  u32x4 kr[S::kLoads], vr[S::kLoads];
  auto fetch = [&](uint32_t k0) {
    const unsigned char* kp = reinterpret_cast<const unsigned char*>(kb + k0 * a.ld_kv);
    const unsigned char* vp = reinterpret_cast<const unsigned char*>(vb + k0 * a.ld_kv);
    const bool whole = k0 + BN <= len;
    const uint32_t last = whole ? BN - 1 : len - 1 - k0;
#pragma unroll
    for (int i = 0; i < S::kLoads; i++) {
      const uint32_t e = i * kPkNT + tid;
      const uint64_t off = (static_cast<uint64_t>(min(e / S::kChunks, last)) * a.ld_kv +
                            min(e % S::kChunks * 8, hd - 8)) * 2;
      kr[i] = *reinterpret_cast<const u32x4*>(kp + off);
      vr[i] = *reinterpret_cast<const u32x4*>(vp + off);
    }
    if (!whole) {  // keys past the end: K repeats the last (and is masked), V is 0
#pragma unroll
      for (int i = 0; i < S::kLoads; i++)
        if ((i * kPkNT + tid) / S::kChunks > last) vr[i] = u32x4{0, 0, 0, 0};
    }
  };
  fetch(0);  // (on its way while q is read)

  // this row's q: operand B of the score product
  half8 qh[S::kStepsQK], ql[HALF ? 1 : S::kStepsQK];
  float c = a.scale;  // scores times c are in log2 units
  if constexpr (HALF) {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (base + tok) * a.ld_q + static_cast<size_t>(head) * hd;
#pragma unroll
    for (int s = 0; s < S::kStepsQK; s++) {
      const uint32_t d = s * 16 + h * 8;
      u32x4 w = {0, 0, 0, 0};
      if (d < hd) w = *reinterpret_cast<const u32x4*>(qp + d);
      qh[s] = __builtin_bit_cast(half8, w);
    }
  } else {
    const float* qp = static_cast<const float*>(a.q) + (base + tok) * a.ld_q + static_cast<size_t>(head) * hd;
    float amax = 0.0f;
#pragma unroll
    for (int s = 0; s < S::kStepsQK; s++) {
      const uint32_t d = s * 16 + h * 8;
      if (d < hd) {
        const float4 x = *reinterpret_cast<const float4*>(qp + d), y = *reinterpret_cast<const float4*>(qp + d + 4);
        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
      }
    }
    amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
    const float f = row_factor(amax);
#pragma unroll
    for (int s = 0; s < S::kStepsQK; s++) {
      const uint32_t d = s * 16 + h * 8;
      float x[8] = {};
      if (d < hd) {
        const float4 u = *reinterpret_cast<const float4*>(qp + d), w = *reinterpret_cast<const float4*>(qp + d + 4);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        _Float16 xh, xl;
        split_half(x[j] * f * a.scale, xh, xl);
        qh[s][j] = xh;
        ql[s][j] = xl;
      }
    }
    c = 1.0f / f;  // a power of two: exact
  }

  f32x16 o[S::kDimBlocks];
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[mb][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;  // kept maximum (log2 units) and this lane's share of the sum

  for (uint32_t k0 = 0; k0 <= tok_last_wg; k0 += BN) {
    // Where the tile reaches past some row's token, a V value that is not
    // finite must not meet that row's zero probability: such values stay out
    // of the tile and are added below to the rows that see them.
    const bool diagonal = k0 + BN - 1 > tok_first_wg;
    bool odd = false;
    if (diagonal) {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < S::kLoads; i++) bits |= odd_halves(vr[i]);
      odd = __syncthreads_or((bits & kOddBits) != 0);  // (also: every wave is done with the tile before)
      if (odd) {
#pragma unroll
        for (int i = 0; i < S::kLoads; i++) vr[i] = only_finite(vr[i]);
      }
    } else {
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < S::kLoads; i++) {
      const int e = i * kPkNT + tid;
      const int r = e / S::kChunks, d = (e % S::kChunks) * 8;
      *reinterpret_cast<u32x4*>(s_k + r * S::kLdK + d) = kr[i];
      *reinterpret_cast<u32x4*>(s_v + r * S::kLdV + d) = vr[i];
    }
    __syncthreads();
    if (k0 + BN <= tok_last_wg) fetch(k0 + BN);
    if (k0 > tok_last) continue;  // (the wave's rows see nothing of this tile)

    // scores
    f32x16 s[S::kKeyBlocks];
#pragma unroll
    for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[b][i] = 0.0f;
#pragma unroll
    for (int t = 0; t < S::kStepsQK; t++)
#pragma unroll
      for (int b = 0; b < S::kKeyBlocks; b++) {
        const half8 kf = *reinterpret_cast<const half8*>(s_k + (b * 32 + n) * S::kLdK + t * 16 + h * 8);
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[t], s[b], 0, 0, 0);
        if constexpr (!HALF) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[t], s[b], 0, 0, 0);
      }
    if (k0 + BN - 1 > tok_first) {
      const int lim = static_cast<int>(tok - k0) - 4 * h;  // keys of this half up to the row's token
#pragma unroll
      for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (b * 32 + 8 * (i / 4) + i % 4 > lim) s[b][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[b][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c;
    if (__any(mx > m + kLag)) {
      const float mn = fmaxf(m, mx), al = exp2_hw(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[mb][i] *= al;
    }
    const float ms = HALF ? m : m - kPShift;
#pragma unroll
    for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        s[b][i] = exp2_hw(fmaf(s[b][i], c, -ms));
        l += s[b][i];
      }
    // values
#pragma unroll
    for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        half8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if constexpr (HALF) {
            ph[j] = static_cast<_Float16>(s[b][t * 8 + j]);
          } else {
            _Float16 xh, xl;
            split_half(s[b][t * 8 + j], xh, xl);
            ph[j] = xh;
            pl[j] = xl;
          }
        }
        const uint16_t* vp = s_v + (b * 32 + t * 16 + 4 * h + ((lane & 15) >> 2)) * S::kLdV +
                             ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++) {
          const half8 vf = join(lds_read_tr(vp + mb * 32), lds_read_tr(vp + 8 * S::kLdV + mb * 32));
          o[mb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph, o[mb], 0, 0, 0);
          if constexpr (!HALF) o[mb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl, o[mb], 0, 0, 0);
        }
      }
    if (odd) {  // rare: the values left out, for the rows that see them (any weight gives the same result)
      for (uint32_t r = k0; r < min(k0 + BN, len); r++) {
        if (r > tok) break;
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const uint32_t d = mb * 32 + 8 * g + 4 * h;
            if (d >= hd) continue;
            const half4 x = *reinterpret_cast<const half4*>(vb + r * a.ld_kv + d);
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float v = static_cast<float>(x[j]);
              o[mb][4 * g + j] += fabsf(v) < INFINITY ? 0.0f : v;
            }
          }
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (row_w + n >= rows) return;
  const float inv = 1.0f / l;
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const uint32_t d = mb * 32 + 8 * g + 4 * h;
      if (d >= hd) continue;
      const size_t at = (base + tok) * a.ld_out + static_cast<size_t>(head) * hd + d;
      if constexpr (HALF) {
        half4 y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = static_cast<_Float16>(o[mb][4 * g + j] * inv);
        *reinterpret_cast<half4*>(static_cast<uint16_t*>(a.out) + at) = y;
      } else {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
            make_float4(o[mb][4 * g] * inv, o[mb][4 * g + 1] * inv, o[mb][4 * g + 2] * inv, o[mb][4 * g + 3] * inv);
      }
    }
}

template <int HDP, int BN>
void launch_shape(const PackedArgs& a, bool half, uint32_t tiles, hipStream_t s) {
  const dim3 grid(tiles * a.n_kv);
  if (half)
    hipLaunchKernelGGL((packed_kernel<HDP, BN, true>), grid, dim3(kPkNT), 0, s, a);
  else
    hipLaunchKernelGGL((packed_kernel<HDP, BN, false>), grid, dim3(kPkNT), 0, s, a);
}

}  // namespace

int launch_attention_packed(const void* q, const uint16_t* k, const uint16_t* v, bool half, const size_t* seq_lens,
                            size_t n_seq, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t ld_q,
                            size_t ld_kv, size_t ld_out, void* out, hipStream_t s) {
  PackedArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.ld_q = ld_q;
  a.ld_kv = ld_kv;
  a.ld_out = ld_out;
  a.n_kv = static_cast<uint32_t>(n_kv_heads);
  a.group = static_cast<uint32_t>(n_heads / n_kv_heads);
  a.hd = static_cast<uint32_t>(head_dim);
  a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(head_dim)));
  struct Seq {
    size_t start, len;
  };
  std::vector<Seq> seqs;
  size_t at = 0;
  for (size_t i = 0; i < n_seq; i++) {
    if (seq_lens[i]) seqs.push_back({at, seq_lens[i]});
    at += seq_lens[i];
  }
  // the longest first: a workgroup's work grows with its place in its sequence
  std::stable_sort(seqs.begin(), seqs.end(), [](const Seq& x, const Seq& y) { return x.len > y.len; });
  const size_t most = 0x7fffffffu / n_kv_heads;  // tiles of one grid
  for (size_t i = 0; i < seqs.size();) {
    size_t tiles = 0;
    a.n_seq = 0;
    while (i < seqs.size() && a.n_seq < kTableSeqs) {
      const size_t t = (seqs[i].len * a.group + kPkRows - 1) / kPkRows;
      if (a.n_seq && tiles + t > most) break;
      a.start[a.n_seq] = static_cast<uint32_t>(seqs[i].start);
      a.len[a.n_seq] = static_cast<uint32_t>(seqs[i].len);
      a.tile0[a.n_seq++] = static_cast<uint32_t>(tiles);
      tiles += t;
      i++;
    }
    const uint32_t t = static_cast<uint32_t>(tiles);
    if (head_dim <= 64)
      launch_shape<64, 64>(a, half, t, s);
    else if (head_dim <= 96)
      launch_shape<96, 64>(a, half, t, s);
    else if (head_dim <= 128)
      launch_shape<128, 64>(a, half, t, s);
    else if (head_dim <= 192)
      launch_shape<192, 64>(a, half, t, s);
    else
      launch_shape<256, 32>(a, half, t, s);
    PRANA_LAUNCH_CHECK();
  }
  return kOk;
}

}  // namespace prana
