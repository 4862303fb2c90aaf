// The 8-bit K/V cache: rows of K and V quantized as they are written
// (prana_kv_write_q8) and read back (prana_kv_read_q8).
//
//   scale = amax / 127 over the values of one KV head in one row (1 when all
//   are 0), i8 = round(x * 127 / amax), ties away from zero, value = i8 * scale.
//
// One scale per row and head, because that is what attention can take out of
// its products: the scale of a K row multiplies its score, that of a V row its
// probability, and the i8 values go to the matrix cores as they are.
//
// Both kernels move each byte once and are bound by memory. Writing, a lane
// holds 8 values of a head (two 16-byte loads of f32, one 8-byte store of i8),
// the lanes of a head find its maximum among them, and a lane takes kItems
// heads whose loads are in flight together. What is read or written once
// passes the caches by (nontemporal); the quantized rows do not, attention
// reads them next.
//
// Measured, 8 heads x 128: K and V rows of four prompts of up to 8191 written in
// 52 us and read back to f32 in 38 (262 MB moved each way, 5.8 TB/s for the two;
// 128 us without the nontemporal accesses and full lines per store), 32767 rows
// to f16 in 32.8 us (6.2 TB/s). A copy reaches 5.0 TB/s, a read alone 6.1. Eight
// or two heads a lane group instead of kItems are slower. One row in each of
// eight sequences: 4 us written, 3 read, the latency of a launch.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "mfma_tile.h"
#include "seq_table.h"
#include "serving.h"

namespace prana {

namespace {

constexpr int kKvNT = 256;
constexpr int kItems = 4;  // heads of a lane group, loads in flight together
// Values a lane writes when a cache is read back.
__host__ __device__ constexpr int read_values(bool half) { return half ? 8 : 4; }

struct KvArgs {
  const void* k;  // the packed side
  const void* v;
  size_t ld;
  uint32_t n_seq, n_kv, hd;
  void* kc[kTableSeqs];
  void* vc[kTableSeqs];
  float* ks[kTableSeqs];
  float* vs[kTableSeqs];
  uint32_t src[kTableSeqs];     // first packed row
  uint32_t rows[kTableSeqs];    // rows to move
  uint32_t first[kTableSeqs];   // first cache row
  uint32_t block0[kTableSeqs];  // first workgroup
};

struct KvSeq {
  void* cache;
  float* scales;
  uint32_t src, rows, first, block0;
};

// The sequence of this workgroup, its K (blockIdx.y 0) or V cache.
__device__ __forceinline__ KvSeq this_seq(const KvArgs& a) {
  const int s = table_find(a.block0, a.n_seq, blockIdx.x);
  const bool second = blockIdx.y != 0;
  return KvSeq{table_at(second ? a.vc : a.kc, s), table_at(second ? a.vs : a.ks, s), table_at(a.src, s),
               table_at(a.rows, s), table_at(a.first, s), table_at(a.block0, s)};
}

// Largest of v over aligned groups of LPH lanes (a power of two).
template <int LPH>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = 1; o < LPH; o <<= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o, 64)));
  return v;
}

// round(|x| * 127 / amax) with ties up, exactly. In f32 the quotient is within
// 127 * 3 * 2^-24 < 2.4e-5 of the real one, so a fraction further than 1e-4
// from a half decides (quantize_fast, whose second result is true otherwise);
// the others (2 values in 10^4) are taken in f64: |x| and amax have 24 bits, so
// a quotient up to 127 that is not a tie is at least 2^-33 from one, while the
// f64 evaluation is off by 2^-43 and the 2^-44 that is added in relative terms
// (2^-37 at most) lifts exact ties over the half.
__device__ __forceinline__ int quantize_fast(float x, float inv, bool& close) {
  const float t = fabsf(x) * inv, u = t + 0.5f, r = floorf(u);
  close = close || fabsf(u - r - 0.5f) > 0.4999f;  // (u is within 1e-4 of a whole number)
  return static_cast<int>(copysignf(r, x));
}
__device__ __forceinline__ int quantize_exact(float x, float amax) {
  const double d = static_cast<double>(fabsf(x)) * 127.0 / static_cast<double>(amax);
  return static_cast<int>(copysignf(static_cast<float>(floor(__fma_rn(d, 0x1p-44, d) + 0.5)), x));
}

template <int LPH>
__global__ __launch_bounds__(kKvNT) void kv_write_kernel(KvArgs a) {
  constexpr int kGroups = kKvNT / LPH;  // heads a workgroup takes at a time
  const KvSeq sq = this_seq(a);
  const float* src = static_cast<const float*>(blockIdx.y ? a.v : a.k);
  int8_t* dst = static_cast<int8_t*>(sq.cache);
  const int sub = threadIdx.x % LPH, grp = threadIdx.x / LPH;
  const bool live = sub * 8u < a.hd;
  const uint64_t n_items = static_cast<uint64_t>(sq.rows) * a.n_kv;
  const uint64_t item0 = static_cast<uint64_t>(blockIdx.x - sq.block0) * (kGroups * kItems) + grp;
  float x[kItems][8];
#pragma unroll
  for (int it = 0; it < kItems; it++) {
    const uint64_t item = item0 + it * kGroups;
    const uint32_t row = static_cast<uint32_t>(item / a.n_kv), head = static_cast<uint32_t>(item % a.n_kv);
#pragma unroll
    for (int j = 0; j < 8; j++) x[it][j] = 0.0f;
    if (item < n_items && live) {
      const f32x4* p = reinterpret_cast<const f32x4*>(src + (static_cast<size_t>(sq.src) + row) * a.ld +
                                                        static_cast<size_t>(head) * a.hd + sub * 8);
      const f32x4 u = __builtin_nontemporal_load(p), w = __builtin_nontemporal_load(p + 1);
      x[it][0] = u.x; x[it][1] = u.y; x[it][2] = u.z; x[it][3] = u.w;
      x[it][4] = w.x; x[it][5] = w.y; x[it][6] = w.z; x[it][7] = w.w;
    }
  }
#pragma unroll
  for (int it = 0; it < kItems; it++) {
    const uint64_t item = item0 + it * kGroups;
    const uint32_t row = static_cast<uint32_t>(item / a.n_kv), head = static_cast<uint32_t>(item % a.n_kv);
    // magnitudes as integers: a NaN is then larger than an infinity
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[it][j]) & 0x7fffffffu);
    top = group_max<LPH>(top);
    const bool finite = top < 0x7f800000u;
    const float amax = __uint_as_float(top);
    float scale = top ? amax / 127.0f : 1.0f;
    const bool fast = amax > 0x1p-100f;  // scale and its inverse are normal numbers
    const float inv = 1.0f / scale;
    if (item >= n_items) continue;
    uint32_t w[2] = {0, 0};
    if (finite && top) {
      bool close = !fast;
#pragma unroll
      for (int j = 0; j < 8; j++)
        w[j / 4] |= static_cast<uint32_t>(quantize_fast(x[it][j], inv, close) & 0xff) << (8 * (j % 4));
      if (close) {
        // (one value after another: unrolled, this branch would be most of the kernel's code)
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = x[it][j];
        w[0] = w[1] = 0;
#pragma unroll 1
        for (int j = 0; j < 8; j++) {
          const uint64_t b = static_cast<uint64_t>(quantize_exact(y[0], amax) & 0xff) << 56;
          const uint64_t v = (static_cast<uint64_t>(w[1]) << 32 | w[0]) >> 8 | b;
          w[0] = static_cast<uint32_t>(v);
          w[1] = static_cast<uint32_t>(v >> 32);
#pragma unroll
          for (int i = 0; i < 7; i++) y[i] = y[i + 1];
        }
      }
    }
    if (!finite) scale = __uint_as_float(0x7fc00000u);  // reads back as NaN
    const size_t r = static_cast<size_t>(sq.first) + row;
    if (live)
      *(device_t<u32x2>*)(dst + (r * a.n_kv + head) * a.hd + sub * 8) = u32x2{w[0], w[1]};
    if (sub == 0) *(device_t<float>*)(sq.scales + r * a.n_kv + head) = scale;
  }
}

// The rows written by kv_write_kernel. A lane moves the values of one 16-byte
// store: 8 halves or 4 floats (a lane of 8 floats would leave its lines half
// written between two stores).
template <int LPH, bool HALF>
__global__ __launch_bounds__(kKvNT) void kv_read_kernel(KvArgs a) {
  constexpr int kGroups = kKvNT / LPH, kPer = read_values(HALF);
  using Word = std::conditional_t<HALF, u32x2, uint32_t>;
  const KvSeq sq = this_seq(a);
  const int8_t* src = static_cast<const int8_t*>(sq.cache);
  void* dst = const_cast<void*>(blockIdx.y ? a.v : a.k);
  const int sub = threadIdx.x % LPH, grp = threadIdx.x / LPH;
  if (sub * static_cast<uint32_t>(kPer) >= a.hd) return;
  const uint64_t n_items = static_cast<uint64_t>(sq.rows) * a.n_kv;
  const uint64_t item0 = static_cast<uint64_t>(blockIdx.x - sq.block0) * (kGroups * kItems) + grp;
  Word w[kItems];
  float scale[kItems];
#pragma unroll
  for (int it = 0; it < kItems; it++) {
    const uint64_t item = item0 + it * kGroups;
    w[it] = Word{};
    scale[it] = 0.0f;
    if (item < n_items) {
      const size_t at = static_cast<size_t>(sq.first) * a.n_kv + item;  // (row, head) of the cache
      w[it] = load_at<Word>(src + at * a.hd + sub * kPer);
      scale[it] = load_at<float>(sq.scales + at);
    }
  }
#pragma unroll
  for (int it = 0; it < kItems; it++) {
    const uint64_t item = item0 + it * kGroups;
    if (item >= n_items) continue;
    const uint32_t row = static_cast<uint32_t>(item / a.n_kv), head = static_cast<uint32_t>(item % a.n_kv);
    const size_t at = (static_cast<size_t>(sq.src) + row) * a.ld + static_cast<size_t>(head) * a.hd + sub * kPer;
    float y[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      uint32_t word;
      if constexpr (HALF)
        word = j < 4 ? w[it].x : w[it].y;
      else
        word = w[it];
      y[j] = static_cast<float>(static_cast<int8_t>(word >> (8 * (j % 4)))) * scale[it];
    }
    if constexpr (HALF) {
      u32x4 h;
#pragma unroll
      for (int j = 0; j < 4; j++)
        h[j] = static_cast<uint32_t>(f32_to_f16(y[2 * j])) | static_cast<uint32_t>(f32_to_f16(y[2 * j + 1])) << 16;
      __builtin_nontemporal_store(h, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(dst) + at));
    } else {
      const f32x4 f = {y[0], y[1], y[2], y[3]};
      __builtin_nontemporal_store(f, reinterpret_cast<f32x4*>(static_cast<float*>(dst) + at));
    }
  }
}

// Lanes of a head: the power of two that holds its pieces of `per` values.
int lanes_per_head(size_t hd, int per) {
  int n = 1;
  while (n * per < static_cast<int>(hd)) n *= 2;
  return n;
}

enum class Move { kWrite, kRead32, kRead16 };

template <int LPH>
void launch_move(Move m, const KvArgs& a, uint32_t blocks, hipStream_t s) {
  const dim3 grid(blocks, 2), nt(kKvNT);
  if (m == Move::kRead32) {
    hipLaunchKernelGGL((kv_read_kernel<LPH, false>), grid, nt, 0, s, a);
  } else if constexpr (LPH <= 32) {
    if (m == Move::kWrite)
      hipLaunchKernelGGL((kv_write_kernel<LPH>), grid, nt, 0, s, a);
    else
      hipLaunchKernelGGL((kv_read_kernel<LPH, true>), grid, nt, 0, s, a);
  }
}

int launch_moves(Move m, const void* k, const void* v, size_t ld, const prana_kv* kv, const size_t* first_rows,
                 const size_t* n_rows, size_t n_seq, size_t n_kv, size_t hd, hipStream_t s) {
  const int lph = lanes_per_head(hd, m == Move::kRead32 ? read_values(false) : 8);
  const size_t per_block = static_cast<size_t>(kKvNT / lph) * kItems;
  KvArgs a{};
  a.k = k;
  a.v = v;
  a.ld = ld;
  a.n_kv = static_cast<uint32_t>(n_kv);
  a.hd = static_cast<uint32_t>(hd);
  size_t src = 0, blocks = 0;
  auto flush = [&]() -> int {
    if (blocks == 0) return kOk;
    const uint32_t b = static_cast<uint32_t>(blocks);
    switch (lph) {
      case 1: launch_move<1>(m, a, b, s); break;
      case 2: launch_move<2>(m, a, b, s); break;
      case 4: launch_move<4>(m, a, b, s); break;
      case 8: launch_move<8>(m, a, b, s); break;
      case 16: launch_move<16>(m, a, b, s); break;
      case 32: launch_move<32>(m, a, b, s); break;
      default: launch_move<64>(m, a, b, s); break;
    }
    PRANA_LAUNCH_CHECK();
    a.n_seq = 0;
    blocks = 0;
    return kOk;
  };
  for (size_t i = 0; i < n_seq; i++) {
    // a launch's lanes fit 32 bits: long sequences go in parts
    constexpr size_t kPartBlocks = size_t{1} << 22;
    const size_t part = std::max<size_t>(1, kPartBlocks * per_block / n_kv);
    for (size_t r = 0; r < n_rows[i]; r += part) {
      const size_t rows = std::min(part, n_rows[i] - r);
      if (a.n_seq == kTableSeqs || blocks > kPartBlocks)
        if (int rc = flush()) return rc;
      const uint32_t e = a.n_seq++;
      a.kc[e] = kv[i].k;
      a.vc[e] = kv[i].v;
      a.ks[e] = kv[i].k_scales;
      a.vs[e] = kv[i].v_scales;
      a.src[e] = static_cast<uint32_t>(src + r);
      a.rows[e] = static_cast<uint32_t>(rows);
      a.first[e] = static_cast<uint32_t>(first_rows[i] + r);
      a.block0[e] = static_cast<uint32_t>(blocks);
      blocks += (rows * n_kv + per_block - 1) / per_block;
    }
    src += n_rows[i];
  }
  return flush();
}

}  // namespace

int launch_kv_write_q8(const float* k, const float* v, size_t ld, const prana_kv* kv, const size_t* first_rows,
                       const size_t* n_rows, size_t n_seq, size_t n_kv_heads, size_t head_dim, hipStream_t s) {
  return launch_moves(Move::kWrite, k, v, ld, kv, first_rows, n_rows, n_seq, n_kv_heads, head_dim, s);
}

int launch_kv_read_q8(const prana_kv* kv, const size_t* first_rows, const size_t* n_rows, size_t n_seq,
                      size_t n_kv_heads, size_t head_dim, bool half, void* k, void* v, size_t ld, hipStream_t s) {
  return launch_moves(half ? Move::kRead16 : Move::kRead32, k, v, ld, kv, first_rows, n_rows, n_seq, n_kv_heads,
                      head_dim, s);
}

}  // namespace prana
