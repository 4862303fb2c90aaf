// Attention of drafted tokens over the caches of several sequences
// (prana_attention_tree). Drafted token i of a sequence whose cache holds
// `past` rows before the drafted ones sees row t when t < past or bit t - past
// of its mask word is set:
//   o_i = sum_t p_it v_t,  p_i = softmax over the seen t of q_i . k_t / sqrt(w).
//
// The rows of a sequence are its (drafted token, query head of the group)
// pairs, so a KV head's cache is read once for all of them. The cache rows are
// split over workgroups; each leaves its rows' maximum, sum and weighted sum,
// which a second launch joins (a sequence that one part holds needs none).
// All products run on the f16 matrix cores: q * log2(e)/sqrt(w), normalised
// per row by a power of two, and the probabilities go in as two halves each
// (22 bits); f16 and i8 cache values are halves exactly. An 8-bit row's K scale
// multiplies its scores, its V scale its probabilities, whose reference then is the
// largest such product.
//
// Two kernels, by the rows of a sequence and KV head:
//   narrow (up to 32 rows): bound by reading the cache. The eight waves of a
//     workgroup share the rows and take different keys, 32 at a time: K goes
//     from memory straight into the operand's registers, V through a corner of
//     LDS that only its wave uses, so no wave waits for another until the end.
//   wide (more rows): bound by the products. Four waves of 32 rows share tiles
//     of 64 or 32 keys in LDS.
// In both S^T = K Q^T leaves a row's scores in the lanes of one column, whose
// registers are, as halves, the operand of O^T += V^T P^T; V comes out of LDS
// transposed to match. The kept maximum lags the scores by up to 2^8 before
// the sums are rescaled, each row's for itself.
//
// Measured, 32/8 heads x 128. Narrow: one token in each of 8 sequences over up
// to 32767 8-bit rows 101 us, 3.9 TB/s of cache (a bare loop over such 128-byte
// pieces of rows reads 5.4); the vector ALU is busy 41 % of the time, half of
// that with turning i8 into halves, the matrix cores 15 %. Twelve waves instead
// of eight spill (110 us); 16-byte loads of i8 gain 0.5 %. Wide: trees of up to
// 64 in 8 sequences over up to 16385 f16 rows 194 to 203 us by card, 365 to 380
// TFLOP/s, twice that with both halves' products (a library's f16 product reaches
// 1155), 11 of it joining; matrix cores busy 45 %, vector ALU 33 %, the rest waits
// for LDS and at barriers. Short calls are launches and trips to memory one after
// another: one token over 511 rows 9 us, four trees of 13 over up to 4099 rows 12.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "mfma_tile.h"
#include "seq_table.h"
#include "serving.h"

namespace prana {

namespace {

constexpr int kTrNT = 256;
constexpr float kLag = 8.0f;
constexpr float kPShift = 7.0f;  // probabilities are kept times 2^7, at most 2^15

struct TreeArgs {
  const float* q;
  const uint64_t* mask;
  float* out;
  float* part;  // [partial row][hd] weighted sums, then [partial row][2] maximum and sum
  size_t part_rows;
  uint32_t n_seq, n_heads, n_kv, group, hd;
  uint32_t whole;           // a cache of up to this many rows is one part
  uint32_t rows_per_split;  // of a longer one
  float scale;  // log2(e) / sqrt(hd)
  const void* k[kTableSeqs];
  const void* v[kTableSeqs];
  const float* ks[kTableSeqs];
  const float* vs[kTableSeqs];
  uint32_t past[kTableSeqs];
  uint32_t tokens[kTableSeqs];
  uint32_t tok0[kTableSeqs];   // first drafted token in q, mask and out
  uint32_t item0[kTableSeqs];  // first work item
  uint32_t part0[kTableSeqs];  // first partial state, in rows (a sequence has tokens * n_heads * splits)
};

struct TreeSeq {
  const void *k, *v;
  const float *ks, *vs;
  uint32_t past, tokens, tok0, item0, part0;
  uint32_t splits;  // parts of the cache rows
};

__device__ __forceinline__ TreeSeq this_seq(const TreeArgs& a, uint32_t item) {
  const int s = table_find(a.item0, a.n_seq, item);
  TreeSeq q{table_at(a.k, s),      table_at(a.v, s),    table_at(a.ks, s),    table_at(a.vs, s),   table_at(a.past, s),
            table_at(a.tokens, s), table_at(a.tok0, s), table_at(a.item0, s), table_at(a.part0, s), 0};
  const uint32_t total = q.past + q.tokens;
  q.splits = total <= a.whole ? 1 : (total + a.rows_per_split - 1) / a.rows_per_split;
  return q;
}

// The mask word of drafted token i, cut to the sequence's tokens.
__device__ __forceinline__ uint64_t mask_word(const TreeArgs& a, const TreeSeq& sq, uint32_t i) {
  const uint64_t own = sq.tokens >= 64 ? ~0ull : (1ull << sq.tokens) - 1;
  return (a.mask ? a.mask[sq.tok0 + i] : (2ull << i) - 1) & own;
}

// Bit j: key first + j is seen (first - past keys lie before the drafted ones).
__device__ __forceinline__ uint64_t seen_from(uint64_t word, int first_minus_past) {
  if (first_minus_past >= 64) return 0;
  if (first_minus_past >= 0) return word >> first_minus_past;
  if (first_minus_past <= -64) return ~0ull;
  return word << -first_minus_past | ((1ull << -first_minus_past) - 1);
}

// Eight i8 values as halves: u = v + 128 in the low bits of 0x6400 is the half
// 1024 + u, and 1152 off that is v.
__device__ __forceinline__ u32x4 i8_to_halves(u32x2 w) {
  const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t b = u[j / 2];
    const uint32_t pair = __builtin_amdgcn_perm(0x64646464u, b, j % 2 ? 0x04030402u : 0x04010400u);
    const half2v x = __builtin_bit_cast(half2v, pair) - half2v{1152.0f16, 1152.0f16};
    o[j] = __builtin_bit_cast(uint32_t, x);
  }
  return u32x4{o[0], o[1], o[2], o[3]};
}

// Eight values of a cache row as loaded, and as halves. Addresses are a
// wave-uniform base, moved from tile to tile, and a lane's 32-bit offset.
template <bool Q8>
struct Piece {
  u32x4 w;
  __device__ __forceinline__ void zero() { w = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void load(const unsigned char* base, uint32_t off) {
    w = load_at<u32x4>(base, off);
  }
  __device__ __forceinline__ u32x4 halves() const { return w; }
};
template <>
struct Piece<true> {
  u32x2 w;
  __device__ __forceinline__ void zero() { w = u32x2{0, 0}; }
  __device__ __forceinline__ void load(const unsigned char* base, uint32_t off) {
    w = load_at<u32x2>(base, off);
  }
  __device__ __forceinline__ u32x4 halves() const { return i8_to_halves(w); }
};

// Four values of a cache row.
template <bool Q8>
__device__ __forceinline__ void load_values(const unsigned char* p, float scale, float* x) {
  if constexpr (Q8) {
    const uint32_t w = load_at<uint32_t>(p);
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = static_cast<float>(static_cast<int8_t>(w >> (8 * j))) * scale;
  } else {
    const half4 v = load_at<half4>(p);
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = static_cast<float>(v[j]);
  }
}

// V scales of 8-bit caches. A row's reference follows the largest product of a
// weight and its V scale among the keys that the row itself sees. The largest
// product then lies between 2^6 and 2^15, where two halves hold 22 bits, whatever
// scales the keys have that the row does not see or gives no weight. With 2^x
// above a key's scale, what is compared is score + x (log2 units); the weights
// and their sum count from the reference, the largest score (m, before c) and
// the rest (e) of it. (8 single tokens over up to 32767 rows, 32/8 x 128: 101 us; 98
// with one power of two for all rows of a wave, over all scales met, where a masked
// row of large scale took the other rows' bits.)
constexpr float kTop = kLag + kPShift;  // products of weights and scales stay under 2^kTop
constexpr float kUnseen = -3e38f;       // in place of a row's reference when it has seen nothing
// The scales themselves are taken times 2^32, so that x reaches from scales of
// 2^-112 to ones past 2^57 (2^64 as values): smaller ones' products are right to
// 2^-137, half steps of 2^-25 over 2^(80 + 32). A scale past 2^96, which only a
// row that nothing sees should have, stops at a float's end.
constexpr float kLift = 0x1p32f;
__device__ __forceinline__ float lifted(float v) {
  return fabsf(v) < INFINITY ? fminf(fmaxf(v * kLift, -0x1.fffffep127f), 0x1.fffffep127f) : v;
}
// x, at least -80: weights stay under 2^(80 + 15), and 2^30 of them under a float's end.
__device__ __forceinline__ float scale_log2(float v) {
  return static_cast<float>(max(static_cast<int>(__float_as_uint(v) >> 23 & 255u) - 126, -80));
}
// A sum of weights, x powers of two up (x <= 0): in two steps, for references that
// lie further apart than a float's range. (Weighted sums of values then vanish
// beside what raised the reference; the weights need not, their scales were small.)
__device__ __forceinline__ float shift_sum(float l, float x) {
  const float half = exp2_hw(0.5f * x);
  return l * half * half;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// ------------------------------------------------------------ narrow: up to 16 RB rows
// Waves of a workgroup: eight, or four of heads whose rows take more than half
// of a unit's registers, one wave to a unit (8 single tokens over up to 30000 f16
// rows, 8/1 x 256: 36.7 us with four, 76 with eight, which spill; 4 over up to
// 200: 12 and 18).
constexpr int narrow_waves(int hdp) { return hdp <= 128 ? 8 : 4; }

template <int HDP>
struct NarrowShape {
  static constexpr int kWaves = narrow_waves(HDP), kNT = 64 * kWaves;
  static constexpr int kRound = 32 * kWaves;  // keys of a workgroup at a time
  static constexpr int kSteps = HDP / 32, kDimBlocks = HDP / 16, kPieces = HDP / 16;
  // V rows an odd multiple of 32 bytes apart: the 32-byte pieces of 8 rows
  // that a transposing read takes at a time fall on different banks
  static constexpr int kLdV = HDP + 16;
  static constexpr int kWaveHalves = 32 * kLdV;
  static constexpr int kLdO = HDP + 4;  // joining the waves: floats per row
  static constexpr int kLdQ = HDP + 8;  // q: 16 rows' reads of 16 bytes on different banks
  static constexpr int kBytes = kWaves * std::max(kWaveHalves * 2, 16 * kLdO * 4);
};

template <int HDP, int RB, bool Q8>
__global__ __launch_bounds__(64 * narrow_waves(HDP), HDP <= 64 && RB == 1 ? 4 : HDP <= 128 ? 2 : 1)
void tree_narrow_kernel(TreeArgs a) {
  using S = NarrowShape<HDP>;
  __shared__ __attribute__((aligned(16))) unsigned char s_mem[S::kBytes];
  __shared__ __attribute__((aligned(16))) uint16_t s_q[2][16 * RB * S::kLdQ];  // the halves of q
  // per wave: K scales of 32 keys, V scales and their scale_log2
  __shared__ __attribute__((aligned(16))) float s_scale[S::kWaves][96];
  __shared__ float s_c[16 * RB], s_m[S::kWaves][16 * RB], s_l[S::kWaves][16 * RB];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  uint16_t* s_v = reinterpret_cast<uint16_t*>(s_mem) + wave * S::kWaveHalves;
  const uint32_t kvh = blockIdx.x % a.n_kv, item = blockIdx.x / a.n_kv;
  const TreeSeq sq = this_seq(a, item);
  const uint32_t split = item - sq.item0, hd = a.hd;
  const uint32_t rows = sq.tokens * a.group, total = sq.past + sq.tokens;
  const uint32_t kbeg = split * a.rows_per_split, kend = sq.splits == 1 ? total : min(total, kbeg + a.rows_per_split);

  // Pieces past the head's width repeat its last one: q is 0 there for K, and
  // V columns there are never stored.
  constexpr uint32_t kSize = Q8 ? 1 : 2;
  const size_t ld = static_cast<size_t>(a.n_kv) * hd, head = static_cast<size_t>(kvh) * hd;
  const unsigned char* kbase = static_cast<const unsigned char*>(sq.k) + head * kSize;
  const unsigned char* vbase = static_cast<const unsigned char*>(sq.v) + head * kSize;
  Piece<Q8> kr[2][S::kSteps], vr[S::kPieces];  // the next keys, on their way
  float sr = 0.0f;  // lanes 0-31: K scale of key lane; 32-63: V scale of key lane - 32
  const float* const scales = Q8 ? (lane < 32 ? sq.ks : sq.vs) + kvh : nullptr;
  // V first: it is used first. The bases are opaque: added up per lane from
  // tile to tile they would take two registers a piece.
  constexpr uint32_t kRowPieces = HDP / 8;
  constexpr bool kEvenRows = 64 % kRowPieces == 0;  // a wave's pieces are whole rows
  const uint32_t ld32 = static_cast<uint32_t>(ld);
  uint32_t voff[kEvenRows ? 1 : S::kPieces], koff[S::kSteps];
#pragma unroll
  for (int p = 0; p < (kEvenRows ? 1 : S::kPieces); p++)
    voff[p] = ((p * 64u + lane) / kRowPieces * ld32 + min((p * 64u + lane) % kRowPieces * 8, hd - 8)) * kSize;
#pragma unroll
  for (int s = 0; s < S::kSteps; s++) koff[s] = (n * ld32 + min(s * 32u + g * 8, hd - 8)) * kSize;
  auto fetch_v = [&](uint32_t k0) {
    const unsigned char* vp = vbase + k0 * ld * kSize;
    asm("" : "+s"(vp));
    if (k0 + 32 <= kend) {
#pragma unroll
      for (int p = 0; p < S::kPieces; p++)
        vr[p].load(kEvenRows ? vp + p * (64 / kRowPieces) * ld * kSize : vp, voff[kEvenRows ? 0 : p]);
      if constexpr (Q8) sr = load_at<float>(scales + static_cast<size_t>(k0 + (lane & 31u)) * a.n_kv);
    } else {  // keys past the end: V is 0
      const uint32_t last = kend - 1 - k0;
#pragma unroll
      for (int p = 0; p < S::kPieces; p++) {
        const uint32_t e = p * 64u + lane, r = e / kRowPieces;
        vr[p].zero();
        if (r <= last) vr[p].load(vp, (r * ld32 + min(e % kRowPieces * 8, hd - 8)) * kSize);
      }
      if constexpr (Q8) {
        sr = 0.0f;
        if ((lane & 31u) <= last) sr = load_at<float>(scales + static_cast<size_t>(k0 + (lane & 31u)) * a.n_kv);
      }
    }
  };
  auto fetch_k = [&](uint32_t k0) {
    const unsigned char* kp = kbase + k0 * ld * kSize;
    asm("" : "+s"(kp));
    if (k0 + 32 <= kend) {
      // (the offsets are opaque too: addresses added up from hoisted 64-bit ones may
      // share registers with what is loaded, which costs 8 single tokens over up to
      // 32767 8-bit rows 107 us instead of 100)
#pragma unroll
      for (int s = 0; s < S::kSteps; s++) asm("" : "+v"(koff[s]));
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int s = 0; s < S::kSteps; s++) kr[b][s].load(kp + b * 16 * ld * kSize, koff[s]);
    } else {  // keys past the end repeat the last (and are masked)
      const uint32_t last = kend - 1 - k0;
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int s = 0; s < S::kSteps; s++)
          kr[b][s].load(kp, (min(b * 16u + n, last) * ld32 + min(s * 32u + g * 8, hd - 8)) * kSize);
    }
  };
  // wave r reads the rows of block r, before the first keys: loads return in order
  QRow<S::kSteps, 32, 4, false> q;
  if (wave < RB) {
    const uint32_t row = min(wave * 16u + n, rows - 1);
    q.load(a.q, ((static_cast<size_t>(sq.tok0) + row / a.group) * a.n_heads + kvh * a.group + row % a.group) * hd,
           g * 8, hd);
  }
  uint32_t k0 = kbeg + wave * 32;
  if (k0 < kend) {
    fetch_v(k0);
    fetch_k(k0);
  }
  if (wave < RB) {
    half8 qh[S::kSteps], ql[S::kSteps];
    const float f = q.halves(a.scale, g * 8, hd, qh, ql);
    if (g == 0) s_c[wave * 16 + n] = f;
#pragma unroll
    for (int s = 0; s < S::kSteps; s++) {
      *reinterpret_cast<half8*>(s_q[0] + (wave * 16 + n) * S::kLdQ + s * 32 + g * 8) = qh[s];
      *reinterpret_cast<half8*>(s_q[1] + (wave * 16 + n) * S::kLdQ + s * 32 + g * 8) = ql[s];
    }
  }

  float c[RB], m[RB], l[RB], e[RB];  // (m: the kept maximum, of scores before c; e: 8-bit)
  uint64_t word[RB];
  f32x4 o[RB][S::kDimBlocks];
#pragma unroll
  for (int r = 0; r < RB; r++) {
    const uint32_t i = min(r * 16u + n, rows - 1) / a.group;
    word[r] = mask_word(a, sq, i);
    m[r] = -INFINITY;
    l[r] = e[r] = 0.0f;
#pragma unroll
    for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
      for (int j = 0; j < 4; j++) o[r][mb][j] = 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RB; r++) c[r] = s_c[r * 16 + n];
  for (; k0 < kend; k0 += S::kRound) {
    // the next keys follow into the registers as these leave them
    const bool more = k0 + S::kRound < kend;
    float sc = sr;
    const bool edge = k0 + 32 > min(sq.past, kend);  // not every row sees every key
    bool odd = false;
    if constexpr (!Q8) {
      // a V value that is not finite must not meet the zero probability of a
      // row that does not see it: it is left out and added below
      if (edge) {
        uint32_t bits = 0;
#pragma unroll
        for (int p = 0; p < S::kPieces; p++) bits |= odd_halves(vr[p].w);
        odd = __any((bits & kOddBits) != 0);
        if (odd) {
#pragma unroll
          for (int p = 0; p < S::kPieces; p++) vr[p].w = only_finite(vr[p].w);
        }
      }
    }
    if constexpr (Q8) {
      // (so too a V scale: it would make every product with its row NaN)
      if (edge) {
        const bool bad = lane >= 32 && !finite(sc);
        odd = __any(bad);
        if (bad) sc = 0.0f;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the reads of the keys before come first)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < S::kPieces; p++) {
      const int e = p * 64 + lane;
      *reinterpret_cast<u32x4*>(s_v + (e / (HDP / 8)) * S::kLdV + (e % (HDP / 8)) * 8) = vr[p].halves();
    }
    if constexpr (Q8) {
      if (lane >= 32) {
        sc = lifted(sc);
        s_scale[wave][32 + lane] = scale_log2(sc);
      }
      s_scale[wave][lane] = sc;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();

    if (more) fetch_v(k0 + S::kRound);
    f32x4 s[RB][2], s2[RB][2];  // from both halves of q
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[r][b][j] = s2[r][b][j] = 0.0f;
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int t = 0; t < S::kSteps; t++) {
        const half8 kf = __builtin_bit_cast(half8, kr[b][t].halves());
#pragma unroll
        for (int r = 0; r < RB; r++) {
          const uint16_t* qp = s_q[0] + (r * 16 + n) * S::kLdQ + t * 32 + g * 8;
          const half8 qh = *reinterpret_cast<const half8*>(qp);
          const half8 ql = *reinterpret_cast<const half8*>(qp + 16 * RB * S::kLdQ);
          s[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh, s[r][b], 0, 0, 0);
          s2[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql, s2[r][b], 0, 0, 0);
        }
      }
    if (more) fetch_k(k0 + S::kRound);
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
      for (int b = 0; b < 2; b++) s[r][b] += s2[r][b];

    float ks[2][4], vs[2][4], vx[2][4];
    if constexpr (Q8) {
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const float4 x = *reinterpret_cast<const float4*>(&s_scale[wave][b * 16 + 4 * g]);
        const float4 y = *reinterpret_cast<const float4*>(&s_scale[wave][32 + b * 16 + 4 * g]);
        const float4 z = *reinterpret_cast<const float4*>(&s_scale[wave][64 + b * 16 + 4 * g]);
        ks[b][0] = x.x; ks[b][1] = x.y; ks[b][2] = x.z; ks[b][3] = x.w;
        vs[b][0] = y.x; vs[b][1] = y.y; vs[b][2] = y.z; vs[b][3] = y.w;
        vx[b][0] = z.x; vx[b][1] = z.y; vx[b][2] = z.z; vx[b][3] = z.w;
      }
    }
    half8 ph[RB], pl[RB];
#pragma unroll
    for (int r = 0; r < RB; r++) {
      if constexpr (Q8) {
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[r][b][j] *= ks[b][j];
      }
      uint32_t seen = ~0u;  // bit 16 b + j: this row sees key b * 16 + 4g + j
      if (edge) {
        const int first = static_cast<int>(k0 + 4 * g);
        seen = static_cast<uint32_t>(seen_from(word[r], first - static_cast<int>(sq.past)));
        const int left = static_cast<int>(kend) - first;  // keys before the end of this part
        seen &= left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (!(seen >> (b * 16 + j) & 1)) s[r][b][j] = -INFINITY;
      }
      auto row_max = [&](auto of) {  // over the row's keys
        float x = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int j = 0; j < 4; j++) x = fmaxf(x, of(b, j));
        x = fmaxf(x, __shfl_xor(x, 16, 64));
        return fmaxf(x, __shfl_xor(x, 32, 64));
      };
      auto rescale = [&](float al) {
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
          for (int j = 0; j < 4; j++) o[r][mb][j] *= al;
      };
      auto relative = [&](bool far) {  // scores too large for their differences to be taken later
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[r][b][j] -= far ? m[r] : 0.0f;
      };
      float ms;  // what a weight counts from
      if constexpr (Q8) {
        const float mx = row_max([&](int b, int j) { return fmaf(s[r][b][j], c[r], vx[b][j]); });
        ms = m[r] == -INFINITY ? kUnseen : fmaf(m[r], c[r], e[r]);
        if (__any(mx - ms > kTop || coarse(mx))) {
          auto past = [&](int b, int j) { return fmaf(s[r][b][j] - m[r], c[r], vx[b][j]); };
          const bool up = row_max(past) - e[r] > kTop;
          const float mw = m[r], ew = e[r], raw = row_max([&](int b, int j) { return s[r][b][j]; });
          m[r] = up ? fmaxf(mw, raw) : mw;
          e[r] = up ? row_max(past) - kPShift : ew;
          const float x = up ? (mw - m[r]) * c[r] + (ew - e[r]) : 0.0f;
          l[r] = shift_sum(l[r], x);
          rescale(exp2_hw(x));
          const bool far = coarse(m[r] * c[r]) && m[r] != -INFINITY;
          if (__any(far)) relative(far);
          ms = m[r] == -INFINITY ? kUnseen : far ? e[r] : fmaf(m[r], c[r], e[r]);
        }
      } else {
        const float mx = row_max([&](int b, int j) { return s[r][b][j]; });
        float from = m[r];  // times c
        if (__any((mx - m[r]) * c[r] > kLag || coarse(mx * c[r]))) {
          const bool up = (mx - m[r]) * c[r] > kLag;  // (each row for itself)
          const float al = up ? exp2_hw((m[r] - mx) * c[r]) : 1.0f;
          from = m[r] = up ? mx : m[r];
          l[r] *= al;
          rescale(al);
          const bool far = coarse(m[r] * c[r]) && m[r] != -INFINITY;
          if (__any(far)) {
            relative(far);
            from = far ? 0.0f : m[r];
          }
        }
        ms = from == -INFINITY ? 0.0f : fmaf(from, c[r], -kPShift);
      }
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          float p0 = exp2_hw(fmaf(s[r][b][j], c[r], -ms)), p1 = exp2_hw(fmaf(s[r][b][j + 1], c[r], -ms));
          l[r] += p0;
          l[r] += p1;
          if constexpr (Q8) {
            p0 *= vs[b][j];
            p1 *= vs[b][j + 1];
          }
          half2v xh, xl;
          split_pair(p0, p1, xh, xl);
          ph[r][b * 4 + j] = xh.x;
          ph[r][b * 4 + j + 1] = xh.y;
          pl[r][b * 4 + j] = xl.x;
          pl[r][b * 4 + j + 1] = xl.y;
        }
    }
    const uint16_t* vp = s_v + (4 * g + (n >> 2)) * S::kLdV + (n & 3) * 4;
#pragma unroll
    for (int mb = 0; mb < S::kDimBlocks; mb++) {
      const half8 vf = join(lds_read_tr(vp + mb * 16), lds_read_tr(vp + 16 * S::kLdV + mb * 16));
#pragma unroll
      for (int r = 0; r < RB; r++) {
        o[r][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[r], o[r][mb], 0, 0, 0);
        o[r][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[r], o[r][mb], 0, 0, 0);
      }
    }
    if (odd) {  // rare (and opaque: nothing of it is worth a register outside)
      uint32_t last4 = hd - 4;
      asm volatile("" : "+s"(last4));
      for (uint32_t t = k0; t < min(k0 + 32, kend); t++) {
        float scale = 1.0f;
        if constexpr (Q8) {
          scale = load_at<float>(sq.vs + static_cast<size_t>(t) * a.n_kv + kvh);
          if (finite(scale)) continue;
        }
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++) {
          float x[4];
          load_values<Q8>(vbase + (t * ld + min(mb * 16u + 4 * g, last4)) * kSize, scale, x);
#pragma unroll
          for (int r = 0; r < RB; r++) {
            const bool sees = seen_from(word[r], static_cast<int>(t) - static_cast<int>(sq.past)) & 1;
#pragma unroll
            for (int j = 0; j < 4; j++) o[r][mb][j] += sees && !finite(x[j]) ? x[j] : 0.0f;
          }
        }
      }
    }
  }

  // join the waves
#pragma unroll
  for (int r = 0; r < RB; r++) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
    m[r] = m[r] == -INFINITY ? (Q8 ? kUnseen : m[r]) : fmaf(m[r], c[r], e[r]);
    if (g == 0) {
      s_m[wave][r * 16 + n] = m[r];
      s_l[wave][r * 16 + n] = l[r];
    }
  }
  __syncthreads();  // (and every wave is done with its part of s_mem)
  float* s_o = reinterpret_cast<float*>(s_mem);
#pragma unroll
  for (int r = 0; r < RB; r++) {
    if (r) __syncthreads();
    const int i = r * 16 + n;
    float M = s_m[0][i];
#pragma unroll
    for (int w = 1; w < S::kWaves; w++) M = fmaxf(M, s_m[w][i]);
    float f = m[r] == -INFINITY ? 0.0f : exp2_hw(m[r] - M);
    if constexpr (Q8) f *= 1.0f / kLift;
#pragma unroll
    for (int mb = 0; mb < S::kDimBlocks; mb++) {
      // a wave that saw nothing of this row holds zeros
      *reinterpret_cast<float4*>(s_o + (wave * 16 + n) * S::kLdO + mb * 16 + 4 * g) =
          make_float4(o[r][mb][0] * f, o[r][mb][1] * f, o[r][mb][2] * f, o[r][mb][3] * f);
    }
    __syncthreads();
    for (int e = tid; e < 16 * (HDP / 4); e += S::kNT) {
      const int rr = e / (HDP / 4);
      const uint32_t d = (e % (HDP / 4)) * 4, row = r * 16 + rr;
      if (row >= rows || d >= hd) continue;
      float4 y = make_float4(0, 0, 0, 0);
      const int ri = r * 16 + rr;
      float top_m = s_m[0][ri];
#pragma unroll
      for (int w = 1; w < S::kWaves; w++) top_m = fmaxf(top_m, s_m[w][ri]);
      float L = 0.0f;
#pragma unroll
      for (int w = 0; w < S::kWaves; w++) {
        const float4 x = *reinterpret_cast<const float4*>(s_o + (w * 16 + rr) * S::kLdO + d);
        y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
        if constexpr (Q8)
          L += shift_sum(s_l[w][ri], s_m[w][ri] - top_m);
        else if (s_m[w][ri] != -INFINITY)
          L = fmaf(s_l[w][ri], exp2_hw(s_m[w][ri] - top_m), L);
      }
      const size_t qrow = static_cast<size_t>(row / a.group) * a.n_heads + kvh * a.group + row % a.group;
      if (sq.splits == 1) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // (L is 0 where the row sees nothing)
        *reinterpret_cast<float4*>(a.out + (static_cast<size_t>(sq.tok0) * a.n_heads + qrow) * hd + d) =
            make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      } else {
        const size_t pr = sq.part0 + qrow * sq.splits + split;
        *reinterpret_cast<float4*>(a.part + pr * hd + d) = y;
        if (d == 0) {
          float* ml = a.part + a.part_rows * hd + pr * 2;
          ml[0] = top_m;
          ml[1] = L;
        }
      }
    }
  }
}

// ------------------------------------------------------------ wide: 128 rows a workgroup
constexpr int kWideRows = 128;

// Keys of a tile: 64, or 32 of heads wider than 96, whose scores and keys on
// their way would spill with 64 (8 trees of 64 over up to 16385, 32/8 x 128:
// 202 us with 64, 195 with 32; 6 of 48 over up to 9000, 24/6 x 192: 125, 113).
constexpr int wide_keys(int hdp) { return hdp <= 96 ? 64 : 32; }

template <int HDP, int BN>
struct WideShape {
  static constexpr int kStepsQK = HDP / 16, kDimBlocks = HDP / 32, kKeyBlocks = BN / 32;
  static constexpr int kChunks = HDP / 8;
  static constexpr int kLdK = HDP + 8;                             // as in the packed prompts' kernel
  static constexpr int kLdV = HDP % 128 == 96 ? HDP : HDP + 32;
  static constexpr int kLoads = BN * kChunks / kTrNT;
};

template <int HDP, bool Q8>
__global__ __launch_bounds__(kTrNT, HDP <= 128 ? 2 : 1) void tree_wide_kernel(TreeArgs a) {
  constexpr int BN = wide_keys(HDP);
  using S = WideShape<HDP, BN>;
  static_assert(BN * S::kChunks % kTrNT == 0, "a tile is a whole number of pieces per lane");
  __shared__ __attribute__((aligned(16))) uint16_t s_k[BN * S::kLdK];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[BN * S::kLdV];
  __shared__ __attribute__((aligned(16))) float s_scale[3][64];  // K scales, V scales, their scale_log2
  // The smaller halves of q, in LDS where the registers would not hold them (6 trees
  // of 48 over up to 9000 f16 rows, 24/6 x 256: 212 us in registers, 140 in LDS, where
  // 21 registers still spill, 14 of the 8-bit form).
  constexpr bool kLowInLds = HDP > 192;
  __shared__ __attribute__((aligned(16))) half8 s_ql[kLowInLds ? S::kStepsQK * kTrNT : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = lane & 31, h = lane >> 5;
  const uint32_t kvh = blockIdx.x % a.n_kv, item = blockIdx.x / a.n_kv;
  const TreeSeq sq = this_seq(a, item);
  const uint32_t hd = a.hd, rows = sq.tokens * a.group, total = sq.past + sq.tokens;
  const uint32_t row_tiles = (rows + kWideRows - 1) / kWideRows;
  const uint32_t split = (item - sq.item0) / row_tiles, row0 = (item - sq.item0) % row_tiles * kWideRows;
  const uint32_t kbeg = split * a.rows_per_split, kend = sq.splits == 1 ? total : min(total, kbeg + a.rows_per_split);
  const bool idle = row0 + wave * 32 >= rows;  // the wave has no rows: it only stages
  const uint32_t row = min(row0 + wave * 32 + n, rows - 1), i = row / a.group;
  const size_t qrow = static_cast<size_t>(i) * a.n_heads + kvh * a.group + row % a.group;
  const uint64_t word = mask_word(a, sq, i);

  constexpr uint32_t kSize = Q8 ? 1 : 2;
  const size_t ld = static_cast<size_t>(a.n_kv) * hd, head = static_cast<size_t>(kvh) * hd;
  const unsigned char* kbase = static_cast<const unsigned char*>(sq.k) + head * kSize;
  const unsigned char* vbase = static_cast<const unsigned char*>(sq.v) + head * kSize;
  Piece<Q8> kr[S::kLoads], vr[S::kLoads];
  float sc = 0.0f;  // lanes 0..BN-1: K scale of key lane; BN..2BN-1: V scales (the rest repeat them)
  const float* const scales = Q8 ? (tid / BN % 2 == 0 ? sq.ks : sq.vs) + kvh : nullptr;
  auto fetch = [&](uint32_t k0) {
    const unsigned char* kp = kbase + k0 * ld * kSize;
    const unsigned char* vp = vbase + k0 * ld * kSize;
    const bool whole = k0 + BN <= kend;
    const uint32_t last = whole ? BN - 1 : kend - 1 - k0;  // keys past the end repeat the last
    if constexpr (Q8) sc = load_at<float>(scales + static_cast<size_t>(k0 + min(tid % BN + 0u, last)) * a.n_kv);
#pragma unroll
    for (int p = 0; p < S::kLoads; p++) {
      const uint32_t e = p * kTrNT + tid, r = e / S::kChunks;
      const uint32_t off = (min(r, last) * static_cast<uint32_t>(ld) + min(e % S::kChunks * 8, hd - 8)) * kSize;
      kr[p].load(kp, off);
      vr[p].load(vp, off);
    }
    if (!whole) {  // their V is 0 (K's scores are masked)
#pragma unroll
      for (int p = 0; p < S::kLoads; p++)
        if ((p * kTrNT + tid) / S::kChunks > last) vr[p].zero();
      if constexpr (Q8)
        if (tid % BN + 0u > last) sc = 0.0f;
    }
  };
  QRow<S::kStepsQK, 16, 2, false> q;  // before the first keys: loads return in order
  q.load(a.q, (static_cast<size_t>(sq.tok0) * a.n_heads + qrow) * hd, h * 8, hd);
  fetch(kbeg);
  half8 qh[S::kStepsQK], ql[S::kStepsQK];
  const float c = q.halves(a.scale, h * 8, hd, qh, ql);
  if constexpr (kLowInLds) {
#pragma unroll
    for (int t = 0; t < S::kStepsQK; t++) s_ql[t * kTrNT + tid] = ql[t];
  }
  f32x16 o[S::kDimBlocks];
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
    for (int j = 0; j < 16; j++) o[mb][j] = 0.0f;
  float m = -INFINITY, l = 0.0f, e = 0.0f;

  for (uint32_t k0 = kbeg; k0 < kend; k0 += BN) {
    const bool edge = k0 + BN > min(sq.past, kend);
    bool odd = false;  // (as in the narrow kernel)
    if (edge) {
      if constexpr (Q8) {
        const bool bad = tid / BN % 2 == 1 && !finite(sc);
        odd = __syncthreads_or(bad);
        if (bad) sc = 0.0f;
      } else {
        uint32_t bits = 0;
#pragma unroll
        for (int p = 0; p < S::kLoads; p++) bits |= odd_halves(vr[p].w);
        odd = __syncthreads_or((bits & kOddBits) != 0);
        if (odd) {
#pragma unroll
          for (int p = 0; p < S::kLoads; p++) vr[p].w = only_finite(vr[p].w);
        }
      }
    } else {
      __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < S::kLoads; p++) {
      const int e = p * kTrNT + tid;
      const int r = e / S::kChunks, d = (e % S::kChunks) * 8;
      *reinterpret_cast<u32x4*>(s_k + r * S::kLdK + d) = kr[p].halves();
      *reinterpret_cast<u32x4*>(s_v + r * S::kLdV + d) = vr[p].halves();
    }
    if constexpr (Q8) {
      if (tid >= BN) {
        sc = lifted(sc);
        if (tid < 2 * BN) s_scale[2][tid % BN] = scale_log2(sc);
      }
      if (tid < 2 * BN) s_scale[tid / BN][tid % BN] = sc;
    }
    __syncthreads();
    if (k0 + BN < kend) fetch(k0 + BN);
    if (idle) continue;

    f32x16 s[S::kKeyBlocks];
#pragma unroll
    for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
      for (int j = 0; j < 16; j++) s[b][j] = 0.0f;
#pragma unroll
    for (int t = 0; t < S::kStepsQK; t++)
#pragma unroll
      for (int b = 0; b < S::kKeyBlocks; b++) {
        const half8 kf = *reinterpret_cast<const half8*>(s_k + (b * 32 + n) * S::kLdK + t * 16 + h * 8);
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[t], s[b], 0, 0, 0);
        const half8 low = kLowInLds ? s_ql[t * kTrNT + tid] : ql[t];
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, low, s[b], 0, 0, 0);
      }
    if constexpr (!kLowInLds) reads_ahead<S::kStepsQK * S::kKeyBlocks, 2>();
    if constexpr (Q8) {
#pragma unroll
      for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const float4 x = *reinterpret_cast<const float4*>(&s_scale[0][b * 32 + 8 * g + 4 * h]);
          s[b][4 * g] *= x.x;
          s[b][4 * g + 1] *= x.y;
          s[b][4 * g + 2] *= x.z;
          s[b][4 * g + 3] *= x.w;
        }
    }
    uint64_t seen = ~0ull;  // bit j: this row sees key k0 + 4h + j
    if (edge) {
      const int first = static_cast<int>(k0 + 4 * h);
      seen = seen_from(word, first - static_cast<int>(sq.past));
      const int left = static_cast<int>(kend) - first;
      seen &= left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
#pragma unroll
      for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
        for (int j = 0; j < 16; j++)
          if (!(seen >> (b * 32 + 8 * (j / 4) + j % 4) & 1)) s[b][j] = -INFINITY;
    }
    auto row_max = [&](auto of) {  // over the row's keys, of a score and the exponent of its V scale (8-bit)
      float x = -INFINITY;
#pragma unroll
      for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          float4 vx = make_float4(0, 0, 0, 0);
          if constexpr (Q8) vx = *reinterpret_cast<const float4*>(&s_scale[2][b * 32 + 8 * g + 4 * h]);
          const float v4[4] = {vx.x, vx.y, vx.z, vx.w};
#pragma unroll
          for (int j = 0; j < 4; j++) x = fmaxf(x, of(s[b][4 * g + j], v4[j]));
        }
      return fmaxf(x, __shfl_xor(x, 32, 64));
    };
    auto rescale = [&](float al) {
#pragma unroll
      for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[mb][j] *= al;
    };
    auto relative = [&](bool far) {
#pragma unroll
      for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
        for (int j = 0; j < 16; j++) s[b][j] -= far ? m : 0.0f;
    };
    float ms;
    if constexpr (Q8) {  // (as in the narrow kernel)
      const float mx = row_max([&](float score, float x) { return fmaf(score, c, x); });
      ms = m == -INFINITY ? kUnseen : fmaf(m, c, e);
      if (__any(mx - ms > kTop || coarse(mx))) {
        auto past = [&](float score, float x) { return fmaf(score - m, c, x); };
        const bool up = row_max(past) - e > kTop;
        const float mw = m, ew = e, raw = row_max([&](float score, float) { return score; });
        m = up ? fmaxf(mw, raw) : mw;
        e = up ? row_max(past) - kPShift : ew;
        const float x = up ? (mw - m) * c + (ew - e) : 0.0f;
        l = shift_sum(l, x);
        rescale(exp2_hw(x));
        const bool far = coarse(m * c) && m != -INFINITY;
        if (__any(far)) relative(far);
        ms = m == -INFINITY ? kUnseen : far ? e : fmaf(m, c, e);
      }
    } else {
      const float mx = row_max([&](float score, float) { return score; });
      float from = m;
      if (__any((mx - m) * c > kLag || coarse(mx * c))) {
        const bool up = (mx - m) * c > kLag;
        const float al = up ? exp2_hw((m - mx) * c) : 1.0f;
        from = m = up ? mx : m;
        l *= al;
        rescale(al);
        const bool far = coarse(m * c) && m != -INFINITY;
        if (__any(far)) {
          relative(far);
          from = far ? 0.0f : m;
        }
      }
      ms = from == -INFINITY ? 0.0f : fmaf(from, c, -kPShift);
    }
#pragma unroll
    for (int b = 0; b < S::kKeyBlocks; b++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        half8 ph, pl;
#pragma unroll
        for (int gg = 0; gg < 2; gg++) {
          float4 vs = make_float4(1, 1, 1, 1);
          if constexpr (Q8) vs = *reinterpret_cast<const float4*>(&s_scale[1][b * 32 + 16 * t + 8 * gg + 4 * h]);
          const float v4[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const int reg = t * 8 + gg * 4 + j;
            float p0 = exp2_hw(fmaf(s[b][reg], c, -ms)), p1 = exp2_hw(fmaf(s[b][reg + 1], c, -ms));
            l += p0;
            l += p1;
            if constexpr (Q8) {
              p0 *= v4[j];
              p1 *= v4[j + 1];
            }
            half2v xh, xl;
            split_pair(p0, p1, xh, xl);
            ph[gg * 4 + j] = xh.x;
            ph[gg * 4 + j + 1] = xh.y;
            pl[gg * 4 + j] = xl.x;
            pl[gg * 4 + j + 1] = xl.y;
          }
        }
        const uint16_t* vp = s_v + (b * 32 + t * 16 + 4 * h + ((lane & 15) >> 2)) * S::kLdV +
                             ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++) {
          const half8 vf = join(lds_read_tr(vp + mb * 32), lds_read_tr(vp + 8 * S::kLdV + mb * 32));
          o[mb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph, o[mb], 0, 0, 0);
          o[mb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl, o[mb], 0, 0, 0);
        }
      }
    if (odd) {  // rare (and opaque: nothing of it is worth a register outside)
      uint32_t last4 = hd - 4;
      asm volatile("" : "+s"(last4));
      for (uint32_t t = k0; t < min(k0 + BN, kend); t++) {
        float scale = 1.0f;
        if constexpr (Q8) {
          scale = load_at<float>(sq.vs + static_cast<size_t>(t) * a.n_kv + kvh);
          if (finite(scale)) continue;
        }
        if (!(seen_from(word, static_cast<int>(t) - static_cast<int>(sq.past)) & 1)) continue;
#pragma unroll
        for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
          for (int g = 0; g < 4; g++) {
            float x[4];
            load_values<Q8>(vbase + (t * ld + min(mb * 32u + 8 * g + 4 * h, last4)) * kSize, scale, x);
#pragma unroll
            for (int j = 0; j < 4; j++) o[mb][4 * g + j] += finite(x[j]) ? 0.0f : x[j];
          }
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  m = m == -INFINITY ? (Q8 ? kUnseen : m) : fmaf(m, c, e);
  if (row0 + wave * 32 + n >= rows) return;
  float f;
  float* dst;
  if (sq.splits == 1) {
    f = l == 0.0f ? 0.0f : 1.0f / l;
    dst = a.out + (static_cast<size_t>(sq.tok0) * a.n_heads + qrow) * hd;
  } else {
    const size_t pr = sq.part0 + qrow * sq.splits + split;
    f = 1.0f;
    dst = a.part + pr * hd;
    if (h == 0) {
      float* ml = a.part + a.part_rows * hd + pr * 2;
      ml[0] = m;
      ml[1] = l;
    }
  }
  constexpr float kDown = Q8 ? 1.0f / kLift : 1.0f;
#pragma unroll
  for (int mb = 0; mb < S::kDimBlocks; mb++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const uint32_t d = mb * 32 + 8 * g + 4 * h;
      if (d < hd)
        *reinterpret_cast<float4*>(dst + d) = make_float4(o[mb][4 * g] * kDown * f, o[mb][4 * g + 1] * kDown * f,
                                                          o[mb][4 * g + 2] * kDown * f, o[mb][4 * g + 3] * kDown * f);
    }
}

// ------------------------------------------------------------ joining the parts
struct JoinArgs {
  const float* part;
  size_t part_rows;
  float* out;
  uint32_t n_seq, n_rows, hd;
  bool q8;                     // the parts' references: of an 8-bit cache (shift_sum)
  uint32_t row0[kTableSeqs];  // first (token, head) row of the sequence in this launch
  uint32_t out0[kTableSeqs];  // its first row of out
  uint32_t splits[kTableSeqs];
  uint32_t part0[kTableSeqs];
};

// A row: M = max m_s, out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), by
// T lanes (a wave, or a workgroup where a row has many parts). A part's row is
// read by LANES lanes, 16 bytes each, T / LANES parts at a time; kBatch loads
// of a lane are in flight together, the first ones before M is known. (Parts of
// 20000 rows, one token, 12/4 x 128: a wave a row 16.5 us for the whole call, a
// workgroup 14.9; up to 16 parts the two take the same.)
template <int T, int LANES>
__global__ __launch_bounds__(256) void tree_join_kernel(JoinArgs a) {
  constexpr int kBatch = 8, kPG = T / LANES, kWaves = T / 64;
  const uint32_t r = blockIdx.x * (256 / T) + __builtin_amdgcn_readfirstlane(threadIdx.x / T);
  const uint32_t tid = threadIdx.x % T, lane = threadIdx.x & 63;
  if (r >= a.n_rows) return;  // (whole waves; with T = 256 never)
  const int si = table_find(a.row0, a.n_seq, r);
  const uint32_t row = r - table_at(a.row0, si), ns = table_at(a.splits, si);
  const size_t out_row = static_cast<size_t>(table_at(a.out0, si)) + row;
  const size_t p0 = table_at(a.part0, si) + static_cast<size_t>(row) * ns;
  const float2* ml = reinterpret_cast<const float2*>(a.part + a.part_rows * a.hd) + p0;
  const uint32_t d = (tid % LANES) * 4, s0 = tid / LANES;
  const float* src = a.part + p0 * a.hd + min(d, a.hd - 4);
  float4 x[kBatch];
  float ms[kBatch];
  auto load = [&](uint32_t s) {
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      const uint32_t at = min(s + k * kPG, ns - 1);
      x[k] = *reinterpret_cast<const float4*>(src + static_cast<size_t>(at) * a.hd);
      ms[k] = ml[at].x;
    }
  };
  load(s0);
  float M = -INFINITY;
  for (uint32_t s = lane; s < ns; s += 64) M = fmaxf(M, ml[s].x);
  M = wave_max_f32(M);
  float L = 0.0f;
  for (uint32_t s = lane; s < ns; s += 64) {
    const float2 v = ml[s];
    if (a.q8)
      L += shift_sum(v.y, v.x - M);
    else if (v.x != -INFINITY)
      L = fmaf(v.y, exp2_hw(v.x - M), L);
  }
  for (int o = 32; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
  float4 y = make_float4(0, 0, 0, 0);
  for (uint32_t s = s0; s < ns; s += kBatch * kPG) {
    if (s != s0) load(s);
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      if (s + k * kPG >= ns) continue;
      // a part without a maximum holds zeros (it saw nothing) or NaN (so were all its scores), which stays
      const float f = ms[k] == -INFINITY ? 0.0f : exp2_hw(ms[k] - M);
      y.x = fmaf(x[k].x, f, y.x);
      y.y = fmaf(x[k].y, f, y.y);
      y.z = fmaf(x[k].z, f, y.z);
      y.w = fmaf(x[k].w, f, y.w);
    }
  }
#pragma unroll
  for (int o = LANES; o < 64; o <<= 1) {
    y.x += __shfl_xor(y.x, o, 64);
    y.y += __shfl_xor(y.y, o, 64);
    y.z += __shfl_xor(y.z, o, 64);
    y.w += __shfl_xor(y.w, o, 64);
  }
  if constexpr (kWaves > 1) {
    __shared__ __attribute__((aligned(16))) float4 s_y[kWaves][64];
    s_y[threadIdx.x >> 6][lane] = y;
    __syncthreads();
    y = s_y[0][lane];
#pragma unroll
    for (int w = 1; w < kWaves; w++) {
      const float4 z = s_y[w][lane];
      y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
    }
  }
  if (tid < LANES && d < a.hd) {
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<float4*>(a.out + out_row * a.hd + d) =
        make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
  }
}

template <int T>
void launch_join(const JoinArgs& j, hipStream_t s) {
  const dim3 grid((j.n_rows + 256 / T - 1) / (256 / T)), nt(256);
  if (j.hd <= 64)
    hipLaunchKernelGGL((tree_join_kernel<T, 16>), grid, nt, 0, s, j);
  else if (j.hd <= 128)
    hipLaunchKernelGGL((tree_join_kernel<T, 32>), grid, nt, 0, s, j);
  else
    hipLaunchKernelGGL((tree_join_kernel<T, 64>), grid, nt, 0, s, j);
}

// ------------------------------------------------------------ plan
// Kernel of a sequence, by its rows per KV head. Two blocks of narrow rows only
// over 8-bit caches of heads up to 128 wide, which leave them the registers (9
// spill at 128 all the same): 10 tokens in four sequences, 12/4 x 128, caches up to
// 4000 and 20000, take 16.7 and 28.4 us there and 19.4 and 38.5 on the wide kernel
// (three quarters of it idle), but 17.9 and 34 against 13.6 and 29 in f16.
enum Width { kNarrow16, kNarrow32, kWide, kWidths };
Width width_of(size_t rows, size_t hd, bool q8) {
  return rows <= 16 ? kNarrow16 : rows <= 32 && hd <= 128 && q8 ? kNarrow32 : kWide;
}

struct Plan {
  Width as[kWidths];               // the kernel that a width's sequences run on in this call
  size_t whole[kWidths];           // caches of up to this many rows are one part
  size_t rows_per_split[kWidths];  // of longer ones
  size_t part_rows;
  size_t floats;
  size_t parts(int w, size_t total) const {
    return total <= whole[w] ? 1 : (total + rows_per_split[w] - 1) / rows_per_split[w];
  }
};

// Workgroups that run at once: 256 compute units times those whose registers
// fit one (the kernels' launch bounds).
size_t resident(Width w, size_t hd) {
  const size_t per_cu = w == kWide ? (hd <= 128 ? 2 : 1) : w == kNarrow16 && hd <= 64 ? 2 : 1;
  return 256 * per_cu;
}

// Cache rows of a part, per kernel: the fewest, in whole tiles, that leave no
// more workgroups than run at once (a few left over for a second round would
// take as long as all of the first), and at least one round of a narrow
// workgroup's waves (256 rows) or 128 rows of a wide one's tiles: one token over
// 4000 rows, 12/4 x 128, takes 11.3 us with parts of 256 rows, 12.5 with 512 and
// 17.1 with 1024; 32 tokens over two caches of up to 3000 21.3 with 64, 18.1
// with 128 and 19.7 with 256. Joining parts costs about 3 us, and a narrow round
// 1.9, so two rounds are one part (one token over 511 rows: 8.9 us; three, where
// other sequences of the call have parts: 15.4 against 11.0).
//
// A kernel's launch and its joining cost a call that has sequences of several
// widths about 8 us each, so those of a smaller width go along on the wider
// kernel, most of it idle, while its longest part grows by no more than `along`
// rows for them. One tree of 40 over 1000 rows beside 4 and 16 single tokens, us on
// one kernel and on two, where it would grow to about
//                     256 rows         512              1000
//   f16    32/8 x 64                   25 29   28 29    41 40    46 40
//          32/8 x 128   27 34  29 35   37 44   42 44    59 61    66 62
//          8/1 x 256    39 47  39 48   56 56   56 56    86 72    90 75
//          16/8 x 256   36 44  48 45   57 53   83 54    89 71   139 72
//   8-bit  32/8 x 64    21 30  23 30   30 33   34 33
//          32/8 x 128   30 34  33 35
//          16/8 x 256   40 44  56 45
// (Two blocks of narrow rows beside one, 8-bit, 32/8 x 64 and x 128: up to 1000 and
// 500 rows 22 us on one kernel, 31 on two.)
size_t along(Width wider, size_t hd, bool q8) {
  if (wider == kNarrow32) return hd <= 64 ? 1024 : 512;
  if (q8) return hd <= 64 ? 384 : 192;
  return hd <= 128 ? 768 : 320;
}

Plan make_plan(const size_t* past, const size_t* n_tree, size_t n_seq, size_t n_heads, size_t n_kv, size_t hd,
               bool q8) {
  const size_t group = n_heads / n_kv;
  Plan p{};
  bool has[kWidths] = {};
  for (int w = 0; w < kWidths; w++) p.as[w] = static_cast<Width>(w);
  for (size_t i = 0; i < n_seq; i++)
    if (n_tree[i]) has[width_of(n_tree[i] * group, hd, q8)] = true;
  auto width = [&](size_t i) { return p.as[width_of(n_tree[i] * group, hd, q8)]; };
  auto tiles = [&](size_t i) { return width(i) == kWide ? (n_tree[i] * group + kWideRows - 1) / kWideRows : 1; };
  // The parts of the sequences on kernel w: the rows of the longest.
  auto split = [&](int w) {
    size_t work = 0, longest = 0;  // cache rows times row tiles
    for (size_t i = 0; i < n_seq; i++)
      if (n_tree[i] && width(i) == w) work += (past[i] + n_tree[i]) * tiles(i);
    const size_t round = 32 * narrow_waves(static_cast<int>(hd)), most = resident(static_cast<Width>(w), hd);
    const size_t unit = w == kWide ? 64 : round, least = w == kWide ? 128 : round;
    size_t r = std::max(least, (work * n_kv / most + unit - 1) / unit * unit);
    p.whole[w] = w == kWide ? least : 2 * round;
    for (int tries = 0; tries < 16; tries++) {
      p.rows_per_split[w] = r;
      size_t n = 0;
      longest = 0;
      for (size_t i = 0; i < n_seq; i++) {
        if (!n_tree[i] || width(i) != w) continue;
        const size_t total = past[i] + n_tree[i], parts = p.parts(w, total);
        n += parts * tiles(i);
        longest = std::max(longest, parts > 1 ? r : total);
      }
      if (n * n_kv <= most) break;
      r += std::max(unit, r / 16 / unit * unit);
    }
    return longest;
  };
  int wider = -1;
  size_t longest = 0;
  for (int w = kWide; w >= 0; w--) {
    if (!has[w]) continue;
    if (wider >= 0) {
      p.as[w] = static_cast<Width>(wider);
      const size_t both = split(wider);
      if (both <= longest + along(p.as[w], hd, q8)) {
        longest = both;
        continue;
      }
      p.as[w] = static_cast<Width>(w);
      split(wider);
    }
    wider = w;
    longest = split(w);
  }
  for (size_t i = 0; i < n_seq; i++) {
    if (!n_tree[i]) continue;
    const size_t parts = p.parts(width(i), past[i] + n_tree[i]);
    if (parts > 1) p.part_rows += n_tree[i] * n_heads * parts;
  }
  p.floats = p.part_rows * (hd + 2);
  return p;
}

template <int HDP>
void launch_width(const TreeArgs& a, Width w, bool q8, uint32_t items, hipStream_t s) {
  const dim3 grid(items * a.n_kv), nt(w == kWide ? kTrNT : 64 * narrow_waves(HDP));
  if (w == kNarrow16) {
    if (q8)
      hipLaunchKernelGGL((tree_narrow_kernel<HDP, 1, true>), grid, nt, 0, s, a);
    else
      hipLaunchKernelGGL((tree_narrow_kernel<HDP, 1, false>), grid, nt, 0, s, a);
  } else if (w == kNarrow32) {
    if constexpr (HDP <= 128) hipLaunchKernelGGL((tree_narrow_kernel<HDP, 2, true>), grid, nt, 0, s, a);
  } else {
    if (q8)
      hipLaunchKernelGGL((tree_wide_kernel<HDP, true>), grid, nt, 0, s, a);
    else
      hipLaunchKernelGGL((tree_wide_kernel<HDP, false>), grid, nt, 0, s, a);
  }
}

}  // namespace

// No plan needs more, and more of anything needs no less: a server allocates for
// its largest sizes once. (The plans themselves do not grow with the cache: longer
// caches are cut into longer parts.) A sequence has at most as many parts as the
// shortest ones make, 128 rows, or a narrow round where no width present is wider;
// and in the launches of one width the parts make at most 2 resident() workgroups,
// each with a tile of rows: a part has at least work / resident() rows, and who has
// parts has more rows than one.
size_t attention_tree_floats(const size_t* past, const size_t* n_tree, size_t n_seq, size_t n_heads,
                             size_t n_kv_heads, size_t head_dim) {
  const size_t group = n_heads / n_kv_heads;
  int widest = kNarrow16;
  for (size_t i = 0; i < n_seq; i++)
    if (n_tree[i]) widest = std::max<int>(widest, width_of(n_tree[i] * group, head_dim, false));
  const bool narrow = widest == kNarrow16;
  const size_t round = 32 * narrow_waves(static_cast<int>(head_dim));
  const size_t least = narrow ? round : 128, whole = narrow ? 2 * round : least;
  size_t most = 0, rows = 0;
  const size_t tile[kWidths] = {16, 32, kWideRows};
  for (int w = 0; w <= widest; w++) most += 2 * resident(static_cast<Width>(w), head_dim) * tile[w];
  for (size_t i = 0; i < n_seq; i++) {
    const size_t total = past[i] + n_tree[i];
    if (total > whole) rows += n_tree[i] * n_heads * ((total + least - 1) / least);
  }
  return std::min(most, rows) * (head_dim + 2);
}

int launch_attention_tree(const float* q, bool q8, const prana_kv* kv, const size_t* past, const size_t* n_tree,
                          size_t n_seq, const uint64_t* mask, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                          float* out, float* workspace, size_t workspace_floats, hipStream_t s) {
  const Plan plan = make_plan(past, n_tree, n_seq, n_heads, n_kv_heads, head_dim, q8);
  if (plan.floats > workspace_floats) return fail(kErrInvalid, "attention_tree: a plan passes its bound");
  TreeArgs a{};
  a.q = q;
  a.mask = mask;
  a.out = out;
  a.part = workspace;
  a.part_rows = plan.part_rows;
  a.n_heads = static_cast<uint32_t>(n_heads);
  a.n_kv = static_cast<uint32_t>(n_kv_heads);
  a.group = static_cast<uint32_t>(n_heads / n_kv_heads);
  a.hd = static_cast<uint32_t>(head_dim);
  a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(head_dim)));
  JoinArgs j{};
  j.part = workspace;
  j.part_rows = plan.part_rows;
  j.out = out;
  j.hd = a.hd;
  j.q8 = q8;
  size_t part0 = 0;
  for (int w = 0; w < kWidths; w++) {
    a.whole = static_cast<uint32_t>(plan.whole[w]);
    a.rows_per_split = static_cast<uint32_t>(std::min<size_t>(plan.rows_per_split[w], 0x7fffffff));
    size_t tok0 = 0, items = 0, most_splits = 0;
    auto flush = [&]() -> int {
      if (a.n_seq) {
        const uint32_t it = static_cast<uint32_t>(items);
        if (head_dim <= 64)
          launch_width<64>(a, static_cast<Width>(w), q8, it, s);
        else if (head_dim <= 96)
          launch_width<96>(a, static_cast<Width>(w), q8, it, s);
        else if (head_dim <= 128)
          launch_width<128>(a, static_cast<Width>(w), q8, it, s);
        else if (head_dim <= 192)
          launch_width<192>(a, static_cast<Width>(w), q8, it, s);
        else
          launch_width<256>(a, static_cast<Width>(w), q8, it, s);
        PRANA_LAUNCH_CHECK();
      }
      if (j.n_seq) {
        if (most_splits > 16)
          launch_join<256>(j, s);
        else
          launch_join<64>(j, s);
        PRANA_LAUNCH_CHECK();
      }
      a.n_seq = j.n_seq = j.n_rows = 0;
      items = most_splits = 0;
      return kOk;
    };
    for (size_t i = 0; i < n_seq; tok0 += n_tree[i], i++) {
      if (!n_tree[i]) continue;
      const size_t rows = n_tree[i] * a.group;
      if (plan.as[width_of(rows, head_dim, q8)] != w) continue;
      const size_t splits = plan.parts(w, past[i] + n_tree[i]);
      if (a.n_seq == kTableSeqs)
        if (int rc = flush()) return rc;
      const uint32_t e = a.n_seq++;
      a.k[e] = kv[i].k;
      a.v[e] = kv[i].v;
      a.ks[e] = kv[i].k_scales;
      a.vs[e] = kv[i].v_scales;
      a.past[e] = static_cast<uint32_t>(past[i]);
      a.tokens[e] = static_cast<uint32_t>(n_tree[i]);
      a.tok0[e] = static_cast<uint32_t>(tok0);
      a.item0[e] = static_cast<uint32_t>(items);
      a.part0[e] = static_cast<uint32_t>(part0);
      items += splits * (w == kWide ? (rows + kWideRows - 1) / kWideRows : 1);
      if (splits > 1) {
        most_splits = std::max(most_splits, splits);
        const uint32_t f = j.n_seq++;
        j.row0[f] = j.n_rows;
        j.out0[f] = static_cast<uint32_t>(tok0 * n_heads);
        j.splits[f] = static_cast<uint32_t>(splits);
        j.part0[f] = static_cast<uint32_t>(part0);
        j.n_rows += static_cast<uint32_t>(n_tree[i] * n_heads);
        part0 += n_tree[i] * n_heads * splits;
      }
    }
    if (int rc = flush()) return rc;
  }
  return kOk;
}

}  // namespace prana
