// Causal attention of whole prompts packed behind one another
// (prana_attention_packed): per sequence and head
//   o_i = sum_{j <= i} p_ij v_j,  p_i = softmax_j(q_i . k_j / sqrt(w)).
//
// One pass over the keys with a running maximum and sum, on the f16 matrix
// cores. The rows of a sequence are its (token, query head of the group)
// pairs, so the heads that share a KV head share its tiles too; a workgroup
// takes 128 rows (32 per wave) and walks the keys up to its last token in
// tiles of 64 or 32, staged through registers into LDS while the tile before is
// computed; where few rows leave the walk over the keys as the bound, groups of
// waves take a workgroup's tiles in turn. Per tile and wave, with 32x32x16 products:
//   S^T = K Q^T : a lane holds one row's scores, 16 of each 32 keys, so the
//                 maximum and sum of a row are taken inside two lanes;
//   O^T += V^T P^T : the scores' registers are, as halves, the operand of
//                 this product (its keys in the order the registers hold
//                 them), and V comes out of LDS transposed to match. No
//                 probability moves between lanes.
// The maximum lags: a row's is raised, and its sums rescaled, only when a score
// passes it by more than 2^8, so probabilities are at most 256.
//
// f32 form: q * log2(e)/sqrt(w), normalised per row by a power of two, and the
// probabilities go in as two halves each (22 bits), twice the products. The
// f16 form rounds a probability to one half (2^-11), as its result is: against 64
// bits its results are off by 2.5e-4 (4 prompts up to 1025, 8/1 x 256) and 2.7e-4
// (2 up to 8191, 32/8 x 128) of their norm, where rounding the result alone makes
// 2.0e-4. Probabilities in two halves would leave that, for 41.3 us instead of 37.6
// and 1075 instead of 810; a caller who wants them has the f32 form.
//
// Measured: two prompts of up to 8191, 32/8 x 128, f16: 810 to 840 us by card, 855
// to 885 TFLOP/s (a library's f16 product reaches 1155; both run at 1.5 to 1.7 GHz);
// matrix cores busy 45 % and vector ALU 41 % of the cycles, seldom both. Nine of up
// to 1501, 14/2 x 64, f32: 52.5 us, 310 TFLOP/s, twice that with both halves' products.
// Computing scores a tile ahead (1044 us instead of 806) and groups of waves that
// take products and softmax in turn (904 instead of 827) cost more registers and
// barriers than they hide.
#include <algorithm>
#include <cmath>
#include <vector>

#include "common.h"
#include "mfma_tile.h"
#include "seq_table.h"
#include "serving.h"

namespace prana {

namespace {

constexpr float kLag = 8.0f;   // how far (log2) scores may pass the kept maximum
constexpr float kPShift = 7.0f;  // probabilities are kept times 2^7 (at most 2^15), so that a half (the smaller
                                 // half of two) resolves 2^-32 of the largest

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
template <int HDP, int BN, int NT>
struct PkShape {
  static constexpr int kStepsQK = HDP / 16, kDimBlocks = HDP / 32, kKeyBlocks = BN / 32;
  static constexpr int kChunks = HDP / 8;  // 16-byte pieces of a row
  // K rows 16 bytes apart from a multiple of 32: the 16-byte reads of 8 rows
  // fall on different banks. V rows 64 bytes (mod 256) apart: so do the
  // 64-byte pieces of 4 rows that a transposing read takes.
  static constexpr int kLdK = HDP + 8;
  static constexpr int kLdV = HDP % 128 == 96 ? HDP : HDP + 32;
  static constexpr int kLoads = BN * kChunks / NT;  // 16-byte pieces a lane stages of K (and of V)
  static constexpr int kTile = BN * (kLdK + kLdV);  // halves of a tile of K and V
  static constexpr int kLdO = HDP + 4;              // joining groups of waves: floats per row
};

// The pieces of K and V rows k0 .. k0+BN-1 (of len) that a lane stages.
// Addresses: a uniform base per tile and piece, and a lane's 32-bit offset that
// stays (the base is opaque: added up per lane from tile to tile the addresses
// would take two registers a piece and as many additions). Pieces past the
// head's width repeat its last one (q is 0 there for K, and V columns there
// are never stored).
template <int BN, int CHUNKS, int NT>
struct TileFetch {
  static constexpr int kLoads = BN * CHUNKS / NT;
  static constexpr bool kEven = NT % CHUNKS == 0;  // a group's pieces are whole rows
  const unsigned char *kb, *vb;
  size_t ld;  // bytes
  uint32_t len, hd, tid;
  uint32_t off[kEven ? 1 : kLoads];
  __device__ __forceinline__ uint32_t offset(uint32_t e, uint32_t last) const {
    return min(e / CHUNKS, last) * static_cast<uint32_t>(ld) + min(e % CHUNKS * 8, hd - 8) * 2;
  }
  __device__ __forceinline__ TileFetch(const uint16_t* k, const uint16_t* v, size_t ld_, uint32_t len_, uint32_t hd_,
                                       uint32_t tid_)
      : kb(reinterpret_cast<const unsigned char*>(k)), vb(reinterpret_cast<const unsigned char*>(v)), ld(ld_ * 2),
        len(len_), hd(hd_), tid(tid_) {
#pragma unroll
    for (int i = 0; i < (kEven ? 1 : kLoads); i++) off[i] = offset(i * NT + tid, BN);
  }
  __device__ __forceinline__ void operator()(uint32_t k0, u32x4* kr, u32x4* vr) const {
    const unsigned char* kp = kb + k0 * ld;
    const unsigned char* vp = vb + k0 * ld;
    asm("" : "+s"(kp), "+s"(vp));
    if (k0 + BN <= len) {
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const size_t up = kEven ? i * (NT / CHUNKS) * ld : 0;
        kr[i] = load_at<u32x4>(kp + up, off[kEven ? 0 : i]);
        vr[i] = load_at<u32x4>(vp + up, off[kEven ? 0 : i]);
      }
    } else {  // keys past the end: K repeats the last (and is masked), V is 0
      const uint32_t last = len - 1 - k0;
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const uint32_t e = i * NT + tid, at = offset(e, last);
        kr[i] = load_at<u32x4>(kp, at);
        vr[i] = u32x4{0, 0, 0, 0};
        if (e / CHUNKS <= last) vr[i] = load_at<u32x4>(vp, at);
      }
    }
  }
};

// Puts a tile from registers into LDS, when every wave is done with the one
// before. Where the tile reaches past some row's token (`edge`), a V value
// that is not finite must not meet that row's zero probability: such values
// stay out of the tile, and true is returned, for them to be added to the rows
// that see them.
template <int BN, int CHUNKS, int NT, int LD_K, int LD_V>
__device__ __forceinline__ bool stage_tile(uint16_t* s_k, uint16_t* s_v, u32x4* kr, u32x4* vr, int tid, bool edge) {
  constexpr int kLoads = BN * CHUNKS / NT;
  bool odd = false;
  if (edge) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kLoads; i++) bits |= odd_halves(vr[i]);
    odd = __syncthreads_or((bits & kOddBits) != 0);
    if (odd) {
#pragma unroll
      for (int i = 0; i < kLoads; i++) vr[i] = only_finite(vr[i]);
    }
  } else {
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kLoads; i++) {
    const int e = i * NT + tid;
    const int r = e / CHUNKS, d = (e % CHUNKS) * 8;
    *reinterpret_cast<u32x4*>(s_k + r * LD_K + d) = kr[i];
    *reinterpret_cast<u32x4*>(s_v + r * LD_V + d) = vr[i];
  }
  __syncthreads();
  return odd;
}

template <bool HALF>
__device__ __forceinline__ void store4(void* out, size_t at, float a, float b, float c, float d) {
  if constexpr (HALF) {
    // A weighted mean of halves is no larger than they are, but the roundings
    // of its weights (2^-11) can carry one at the end of their range past it.
    auto half = [](float x) {
      return static_cast<_Float16>(fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x);
    };
    const half4 y = {half(a), half(b), half(c), half(d)};
    *reinterpret_cast<half4*>(static_cast<uint16_t*>(out) + at) = y;
  } else {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(a, b, c, d);
  }
}

// Keys of a tile: 64, or 32 in the f32 form of heads wider than 96, which 64
// would make spill (5 prompts up to 700 and 3000, 32/8 x 128: 44 and 663 us with
// 64, 37 and 641 with 32), and where two waves stage a tile of heads wider
// than 64.
constexpr int packed_keys(int hdp, bool half, int waves) {
  return hdp <= 64 || (waves == 4 && (half || hdp <= 96)) ? 64 : 32;
}

// WAVES waves take 32 rows each and share tiles; GROUPS such groups of a
// workgroup take the tiles in turn and join their sums at the end.
template <int HDP, bool HALF, int WAVES, int GROUPS>
__global__ __launch_bounds__(64 * WAVES * GROUPS, GROUPS == 1 && HDP <= 64 ? 3 : 2) void packed_kernel(PackedArgs a) {
  constexpr int NT = 64 * WAVES, BN = packed_keys(HDP, HALF, WAVES), kRows = 32 * WAVES;
  using S = PkShape<HDP, BN, NT>;
  static_assert(BN * S::kChunks % NT == 0, "a tile is a whole number of pieces per lane");
  constexpr int kTiles = GROUPS * S::kTile, kSums = (GROUPS - 1) * kRows * S::kLdO * 2;  // halves
  __shared__ __attribute__((aligned(16))) uint16_t s_tiles[kTiles > kSums ? kTiles : kSums];
  __shared__ float s_ml[GROUPS][2][kRows];
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
  const int tid = threadIdx.x % NT, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint16_t* const s_k = s_tiles + group * S::kTile;
  uint16_t* const s_v = s_k + BN * S::kLdK;
  const int n = lane & 31, h = lane >> 5;
  const uint32_t kvh = blockIdx.x % a.n_kv, tile = blockIdx.x / a.n_kv;
  const int sq = table_find(a.tile0, a.n_seq, tile);
  const uint32_t len = table_at(a.len, sq), rows = len * a.group;
  const uint32_t n_tiles = (rows + kRows - 1) / kRows;
  // the last tiles see the most keys: they go first
  const uint32_t row0 = (n_tiles - 1 - (tile - table_at(a.tile0, sq))) * kRows;
  const size_t base = table_at(a.start, sq);
  const uint32_t row_w = row0 + wave * 32;                       // the wave's first row
  const uint32_t row = min(row_w + n, rows - 1);                 // (rows past the end repeat the last one)
  const uint32_t tok = row / a.group, head = kvh * a.group + row % a.group;
  const uint32_t tok_first_wg = row0 / a.group;
  const uint32_t tok_last_wg = (min(row0 + kRows, rows) - 1) / a.group;
  const uint32_t tok_first = min(row_w, rows - 1) / a.group;      // of the wave
  const uint32_t tok_last = min(row_w + 31, rows - 1) / a.group;
  const uint32_t hd = a.hd;

  QRow<S::kStepsQK, 16, 2, HALF> q;
  q.load(a.q, (base + tok) * a.ld_q + static_cast<size_t>(head) * hd, h * 8, hd);
  const uint16_t* kb = a.k + base * a.ld_kv + static_cast<size_t>(kvh) * hd;
  const uint16_t* vb = a.v + base * a.ld_kv + static_cast<size_t>(kvh) * hd;
  u32x4 kr[S::kLoads], vr[S::kLoads];
  const TileFetch<BN, S::kChunks, NT> fetch(kb, vb, a.ld_kv, len, hd, tid);
  if (group * BN <= tok_last_wg) fetch(group * BN, kr, vr);
  half8 qh[S::kStepsQK], ql[HALF ? 1 : S::kStepsQK];
  const float c = q.halves(a.scale, h * 8, hd, qh, ql);

  f32x16 o[S::kDimBlocks];
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[mb][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;  // kept maximum (of scores before c) and this lane's share of the sum

  constexpr uint32_t kRound = GROUPS * BN;
  for (uint32_t r0 = 0; r0 <= tok_last_wg; r0 += kRound) {
    const uint32_t k0 = r0 + group * BN;
    const bool odd = stage_tile<BN, S::kChunks, NT, S::kLdK, S::kLdV>(s_k, s_v, kr, vr, tid,
                                                                      r0 + kRound - 1 > tok_first_wg);
    if (k0 + kRound <= tok_last_wg) fetch(k0 + kRound, kr, vr);
    if (k0 > tok_last) continue;  // (the wave's rows see nothing of this tile)
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
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    float from = m;  // what scores are taken relative to, times c
    if (__any((mx - m) * c > kLag || coarse(mx * c))) {
      const bool up = (mx - m) * c > kLag;  // (each row for itself)
      const float al = up ? exp2_hw((m - mx) * c) : 1.0f;
      from = m = up ? mx : m;
      l *= al;
#pragma unroll
      for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[mb][i] *= al;
      if (__any(coarse(m * c))) {
        const bool far = coarse(m * c);
        from = far ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
          for (int i = 0; i < 16; i++) s[b][i] -= far ? m : 0.0f;
      }
    }
    const float ms = fmaf(from, c, -kPShift);
#pragma unroll
    for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        half8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float p0 = exp2_hw(fmaf(s[b][t * 8 + j], c, -ms)), p1 = exp2_hw(fmaf(s[b][t * 8 + j + 1], c, -ms));
          l += p0;
          l += p1;
          half2v xh, xl;
          if constexpr (HALF)
            xh = __builtin_convertvector((f32x2{p0, p1}), half2v);
          else
            split_pair(p0, p1, xh, xl);
          ph[j] = xh.x;
          ph[j + 1] = xh.y;
          if constexpr (!HALF) {
            pl[j] = xl.x;
            pl[j + 1] = xl.y;
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
      uint32_t last4 = hd - 4;  // (opaque: nothing of this is worth a register outside)
      asm volatile("" : "+s"(last4));
      for (uint32_t r = k0; r < min(k0 + BN, len); r++) {
        if (r > tok) break;
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const half4 x = *reinterpret_cast<const half4*>(vb + r * a.ld_kv + min(mb * 32u + 8 * g + 4 * h, last4));
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
  if constexpr (GROUPS > 1) {
    m *= c;
    // the other groups leave their sums in LDS, for the first to join
    const int row_wg = wave * 32 + n;
    __syncthreads();
    if (h == 0) {
      s_ml[group][0][row_wg] = m;
      s_ml[group][1][row_wg] = l;
    }
    float* const s_o = reinterpret_cast<float*>(s_tiles) + row_wg * S::kLdO + 4 * h;
    if (group > 0) {
#pragma unroll
      for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
        for (int g = 0; g < 4; g++)
          *reinterpret_cast<float4*>(s_o + (group - 1) * kRows * S::kLdO + mb * 32 + 8 * g) =
              make_float4(o[mb][4 * g], o[mb][4 * g + 1], o[mb][4 * g + 2], o[mb][4 * g + 3]);
    }
    __syncthreads();
    if (group > 0) return;
    // Every row sees the first key, so the first group's maximum is a number (or
    // the row's scores are not). In another group a row's is one from its first
    // tile on: a tile's tokens are whole blocks of rows, so a wave's rows see its
    // first key together.
    const float mine = m;
#pragma unroll
    for (int i = 1; i < GROUPS; i++) m = fmaxf(m, s_ml[i][0][row_wg]);
    const float f0 = exp2_hw(mine - m);
    l *= f0;
#pragma unroll
    for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[mb][i] *= f0;
#pragma unroll
    for (int i = 1; i < GROUPS; i++) {
      const float f = exp2_hw(s_ml[i][0][row_wg] - m);
      l = fmaf(s_ml[i][1][row_wg], f, l);
#pragma unroll
      for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const float4 x = *reinterpret_cast<const float4*>(s_o + (i - 1) * kRows * S::kLdO + mb * 32 + 8 * g);
          o[mb][4 * g] = fmaf(x.x, f, o[mb][4 * g]);
          o[mb][4 * g + 1] = fmaf(x.y, f, o[mb][4 * g + 1]);
          o[mb][4 * g + 2] = fmaf(x.z, f, o[mb][4 * g + 2]);
          o[mb][4 * g + 3] = fmaf(x.w, f, o[mb][4 * g + 3]);
        }
    }
  }
  if (row_w + n >= rows) return;
  const float inv = 1.0f / l;
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const uint32_t d = mb * 32 + 8 * g + 4 * h;
      if (d >= hd) continue;
      store4<HALF>(a.out, (base + tok) * a.ld_out + static_cast<size_t>(head) * hd + d, o[mb][4 * g] * inv,
                   o[mb][4 * g + 1] * inv, o[mb][4 * g + 2] * inv, o[mb][4 * g + 3] * inv);
    }
}

// ------------------------------------------------------------ heads wider than 128
// 32 rows of such heads would fill the registers of a wave that runs alone on
// its unit, with nothing to hide its waits behind. So a wave takes 16 rows
// (16x16x32 products, twice the LDS reads per product) and four waves 64;
// tiles of 32 keys. Such heads often share one KV head, and 64 rows of it are
// few workgroups that walk long prompts alone, so each has two such groups of
// waves, which take the tiles in turn and join their sums at the end. Four
// prompts of up to 1025, 8/1 x 256, f16: 37.3 us, 279 TFLOP/s (32-row waves 59,
// one group of 16-row waves 48); bound by LDS, from which a wave reads every
// operand for 16 rows only.
constexpr int kWideRows = 64, kWideBN = 32, kWideGroups = 2;

template <int HDP>
struct PkWideShape {
  static constexpr int kNT = 4 * kWideRows;  // lanes of a group
  static constexpr int kSteps = HDP / 32, kDimBlocks = HDP / 16, kChunks = HDP / 8;
  static constexpr int kLdK = HDP + 8;
  static constexpr int kLdV = HDP + 16;  // 32-byte pieces of 8 rows on different banks
  static constexpr int kLoads = kWideBN * kChunks / kNT;
  static constexpr int kTile = kWideBN * (kLdK + kLdV);  // halves of a group's K and V
  static constexpr int kLdO = HDP + 4;                   // joining the groups: floats per row
  static_assert((kWideGroups - 1) * kWideRows * kLdO * 4 <= kWideGroups * kTile * 2, "the groups' sums fit the tiles");
};

template <int HDP, bool HALF>
__global__ __launch_bounds__(kWideGroups * 4 * kWideRows, 2) void packed_wide_kernel(PackedArgs a) {
  using S = PkWideShape<HDP>;
  constexpr int NT = S::kNT, kRows = kWideRows, GROUPS = kWideGroups;
  static_assert(kWideBN * S::kChunks % NT == 0, "a tile is a whole number of pieces per lane");
  __shared__ __attribute__((aligned(16))) uint16_t s_tiles[GROUPS * S::kTile];
  __shared__ float s_ml[GROUPS][2][kRows];
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
  const int tid = threadIdx.x % NT, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint16_t* const s_k = s_tiles + group * S::kTile;
  uint16_t* const s_v = s_k + kWideBN * S::kLdK;
  const int n = lane & 15, g = lane >> 4;
  const uint32_t kvh = blockIdx.x % a.n_kv, tile = blockIdx.x / a.n_kv;
  const int sq = table_find(a.tile0, a.n_seq, tile);
  const uint32_t len = table_at(a.len, sq), rows = len * a.group;
  const uint32_t n_tiles = (rows + kRows - 1) / kRows;
  const uint32_t row0 = (n_tiles - 1 - (tile - table_at(a.tile0, sq))) * kRows;
  const size_t base = table_at(a.start, sq);
  const uint32_t row_w = row0 + wave * 16;
  const uint32_t row = min(row_w + n, rows - 1);
  const uint32_t tok = row / a.group, head = kvh * a.group + row % a.group;
  const uint32_t tok_first_wg = row0 / a.group;
  const uint32_t tok_last_wg = (min(row0 + kRows, rows) - 1) / a.group;
  const uint32_t tok_first = min(row_w, rows - 1) / a.group;
  const uint32_t tok_last = min(row_w + 15, rows - 1) / a.group;
  const uint32_t hd = a.hd;

  QRow<S::kSteps, 32, 4, HALF> q;
  q.load(a.q, (base + tok) * a.ld_q + static_cast<size_t>(head) * hd, g * 8, hd);
  const uint16_t* kb = a.k + base * a.ld_kv + static_cast<size_t>(kvh) * hd;
  const uint16_t* vb = a.v + base * a.ld_kv + static_cast<size_t>(kvh) * hd;
  u32x4 kr[S::kLoads], vr[S::kLoads];
  const TileFetch<kWideBN, S::kChunks, NT> fetch(kb, vb, a.ld_kv, len, hd, tid);
  if (group * kWideBN <= tok_last_wg) fetch(group * kWideBN, kr, vr);
  half8 qh[S::kSteps], ql[HALF ? 1 : S::kSteps];
  const float c = q.halves(a.scale, g * 8, hd, qh, ql);

  f32x4 o[S::kDimBlocks];
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
    for (int i = 0; i < 4; i++) o[mb][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  constexpr uint32_t kRound = GROUPS * kWideBN;
  for (uint32_t r0 = 0; r0 <= tok_last_wg; r0 += kRound) {
    const uint32_t k0 = r0 + group * kWideBN;
    const bool odd = stage_tile<kWideBN, S::kChunks, NT, S::kLdK, S::kLdV>(s_k, s_v, kr, vr, tid,
                                                                           r0 + kRound - 1 > tok_first_wg);
    if (k0 + kRound <= tok_last_wg) fetch(k0 + kRound, kr, vr);
    if (k0 > tok_last) continue;  // (the wave's rows see nothing of this tile)

    f32x4 s[2], s2[2];  // (two chains of products each)
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) s[b][i] = s2[b][i] = 0.0f;
#pragma unroll
    for (int t = 0; t < S::kSteps; t++)
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const half8 kf = *reinterpret_cast<const half8*>(s_k + (b * 16 + n) * S::kLdK + t * 32 + g * 8);
        if constexpr (HALF) {
          f32x4& x = t % 2 ? s2[b] : s[b];
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[t], x, 0, 0, 0);
        } else {
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[t], s[b], 0, 0, 0);
          s2[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[t], s2[b], 0, 0, 0);
        }
      }
#pragma unroll
    for (int b = 0; b < 2; b++) s[b] += s2[b];
    if (k0 + kWideBN - 1 > tok_first) {
      const int lim = static_cast<int>(tok - k0) - 4 * g;
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (b * 16 + i > lim) s[b][i] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    float from = m;
    if (__any((mx - m) * c > kLag || coarse(mx * c))) {
      const bool up = (mx - m) * c > kLag;  // (each row for itself)
      const float al = up ? exp2_hw((m - mx) * c) : 1.0f;
      from = m = up ? mx : m;
      l *= al;
#pragma unroll
      for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[mb][i] *= al;
      if (__any(coarse(m * c))) {
        const bool far = coarse(m * c);
        from = far ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[b][i] -= far ? m : 0.0f;
      }
    }
    const float ms = fmaf(from, c, -kPShift);
    half8 ph, pl;
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float p0 = exp2_hw(fmaf(s[b][i], c, -ms)), p1 = exp2_hw(fmaf(s[b][i + 1], c, -ms));
        l += p0;
        l += p1;
        half2v xh, xl;
        if constexpr (HALF)
          xh = __builtin_convertvector((f32x2{p0, p1}), half2v);
        else
          split_pair(p0, p1, xh, xl);
        ph[b * 4 + i] = xh.x;
        ph[b * 4 + i + 1] = xh.y;
        if constexpr (!HALF) {
          pl[b * 4 + i] = xl.x;
          pl[b * 4 + i + 1] = xl.y;
        }
      }
    const uint16_t* vp = s_v + (4 * g + (n >> 2)) * S::kLdV + (n & 3) * 4;
#pragma unroll
    for (int mb = 0; mb < S::kDimBlocks; mb++) {
      const half8 vf = join(lds_read_tr(vp + mb * 16), lds_read_tr(vp + 16 * S::kLdV + mb * 16));
      o[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, o[mb], 0, 0, 0);
      if constexpr (!HALF) o[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[mb], 0, 0, 0);
    }
    if (odd) {  // rare: the values left out, for the rows that see them
      uint32_t last4 = hd - 4;
      asm volatile("" : "+s"(last4));
      for (uint32_t r = k0; r < min(k0 + kWideBN, len); r++) {
        if (r > tok) break;
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++) {
          const uint32_t d = mb * 16 + 4 * g;
          const half4 x = *reinterpret_cast<const half4*>(vb + r * a.ld_kv + min(d, last4));
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float v = static_cast<float>(x[j]);
            o[mb][j] += fabsf(v) < INFINITY ? 0.0f : v;
          }
        }
      }
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  m *= c;
  // the other groups leave their sums in LDS, for the first to join
  const int row_wg = wave * 16 + n;
  float* const s_o = reinterpret_cast<float*>(s_tiles) + row_wg * S::kLdO + 4 * g;
  __syncthreads();
  if (g == 0) {
    s_ml[group][0][row_wg] = m;
    s_ml[group][1][row_wg] = l;
  }
  if (group > 0) {
#pragma unroll
    for (int mb = 0; mb < S::kDimBlocks; mb++)
      *reinterpret_cast<f32x4*>(s_o + (group - 1) * kRows * S::kLdO + mb * 16) = o[mb];
  }
  __syncthreads();
  if (group > 0 || row_w + n >= rows) return;
  // (the maxima are numbers as in the kernel above)
  const float mine = m;
#pragma unroll
  for (int i = 1; i < GROUPS; i++) m = fmaxf(m, s_ml[i][0][row_wg]);
  const float f0 = exp2_hw(mine - m);
  l *= f0;
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++) o[mb] *= f0;
#pragma unroll
  for (int i = 1; i < GROUPS; i++) {
    const float f = exp2_hw(s_ml[i][0][row_wg] - m);
    l = fmaf(s_ml[i][1][row_wg], f, l);
#pragma unroll
    for (int mb = 0; mb < S::kDimBlocks; mb++)
      o[mb] += *reinterpret_cast<const f32x4*>(s_o + (i - 1) * kRows * S::kLdO + mb * 16) * f;
  }
  const float inv = 1.0f / l;
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++) {
    const uint32_t d = mb * 16 + 4 * g;
    if (d < hd) {
      const f32x4 y = o[mb] * inv;
      store4<HALF>(a.out, (base + tok) * a.ld_out + static_cast<size_t>(head) * hd + d, y[0], y[1], y[2], y[3]);
    }
  }
}

struct Seq {
  size_t start, len;
};

// Rows of a workgroup.
size_t tile_rows(size_t head_dim, bool divided) {
  return head_dim > 128 ? kWideRows : divided && head_dim <= 96 ? 64 : 128;
}

size_t tile_lanes(size_t head_dim, bool divided) { return head_dim > 128 || divided ? 512 : 256; }

// Whether workgroups divide the keys among groups of waves: four groups of two
// waves (64 rows) for heads up to 96 wide, two of four for heads up to 128. That
// shortens the longest walk over the keys, which bounds a call of few rows, but
// such a workgroup has a compute unit to itself (and joins its groups, so
// not for short walks: 300 tokens, 8/2 x 128, 12.4 us whole,
// 12.8 divided; 6/6 x 48 8.4, 7.7). In units of a tile of 64 keys
// (1.1 to 1.4 us), the longest walk is len / 64; divided workgroups cost about
// 3 each and 0.45 (0.8 with two groups) per tile of their walks, on 256 units.
// One prompt of 1500, 14/2 x 64, f32: 36 us whole, 22 divided; two of up to
// 3500, 6/6 x 48: 81 and 59; one of 1500, 32/8 x 128: 63 and 52; but eight of up
// to 600, 14/2 x 64: 20 and 25, and one of 3500, 32/8 x 128: 212 and 217.
bool divide(const std::vector<Seq>& seqs, size_t group, size_t n_kv, size_t head_dim) {  // seqs: the longest first
  if (head_dim > 128 || seqs.empty() || seqs[0].len < (head_dim <= 96 ? 256 : 512)) return false;
  const size_t rows = tile_rows(head_dim, true);
  const double per_tile = head_dim <= 96 ? 0.45 : 0.8;
  double cost = 0;
  for (const Seq& q : seqs) {
    const double wgs = static_cast<double>((q.len * group + rows - 1) / rows * n_kv);
    cost += wgs * (3 + per_tile * static_cast<double>(q.len) / 128);  // (half of len on average)
  }
  return cost / 256 < static_cast<double>(seqs[0].len) / 64;
}

template <int HDP, bool HALF>
void launch_shape(const PackedArgs& a, bool divided, uint32_t tiles, hipStream_t s) {
  const dim3 grid(tiles * a.n_kv), lanes(static_cast<uint32_t>(tile_lanes(HDP, divided)));
  if constexpr (HDP <= 128) {
    constexpr int kWaves = HDP <= 96 ? 2 : 4;
    if (divided)
      hipLaunchKernelGGL((packed_kernel<HDP, HALF, kWaves, 8 / kWaves>), grid, lanes, 0, s, a);
    else
      hipLaunchKernelGGL((packed_kernel<HDP, HALF, 4, 1>), grid, lanes, 0, s, a);
  } else {
    hipLaunchKernelGGL((packed_wide_kernel<HDP, HALF>), grid, lanes, 0, s, a);
  }
}

template <int HDP>
void launch_type(const PackedArgs& a, bool half, bool divided, uint32_t tiles, hipStream_t s) {
  if (half)
    launch_shape<HDP, true>(a, divided, tiles, s);
  else
    launch_shape<HDP, false>(a, divided, tiles, s);
}

}  // namespace

// (Workgroups divide the keys for few rows only.)
size_t packed_lanes(size_t len, size_t n_heads, size_t n_kv_heads, size_t head_dim) {
  const size_t rows = tile_rows(head_dim, false);
  return (len * (n_heads / n_kv_heads) + rows - 1) / rows * n_kv_heads * tile_lanes(head_dim, false);
}

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
  std::vector<Seq> seqs;
  size_t at = 0;
  for (size_t i = 0; i < n_seq; i++) {
    if (seq_lens[i]) seqs.push_back({at, seq_lens[i]});
    at += seq_lens[i];
  }
  // the longest first: a workgroup's work grows with its place in its sequence
  std::stable_sort(seqs.begin(), seqs.end(), [](const Seq& x, const Seq& y) { return x.len > y.len; });
  const bool divided = divide(seqs, a.group, n_kv_heads, head_dim);
  const size_t rows = tile_rows(head_dim, divided);
  // Tiles of one grid: its lanes are to fit 32 bits (one sequence's do: packed_lanes).
  const size_t most = (size_t{1} << 22) / n_kv_heads;
  for (size_t i = 0; i < seqs.size();) {
    size_t tiles = 0;
    a.n_seq = 0;
    while (i < seqs.size() && a.n_seq < kTableSeqs) {
      const size_t t = (seqs[i].len * a.group + rows - 1) / rows;
      if (a.n_seq && tiles + t > most) break;
      a.start[a.n_seq] = static_cast<uint32_t>(seqs[i].start);
      a.len[a.n_seq] = static_cast<uint32_t>(seqs[i].len);
      a.tile0[a.n_seq++] = static_cast<uint32_t>(tiles);
      tiles += t;
      i++;
    }
    const uint32_t t = static_cast<uint32_t>(tiles);
    if (head_dim <= 64)
      launch_type<64>(a, half, divided, t, s);
    else if (head_dim <= 96)
      launch_type<96>(a, half, divided, t, s);
    else if (head_dim <= 128)
      launch_type<128>(a, half, divided, t, s);
    else if (head_dim <= 192)
      launch_type<192>(a, half, divided, t, s);
    else
      launch_type<256>(a, half, divided, t, s);
    PRANA_LAUNCH_CHECK();
  }
  return kOk;
}

}  // namespace prana
