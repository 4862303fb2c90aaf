// The sequences of one launch, as arrays in its kernel arguments with one
// entry per lane. A wave finds its sequence and reads everything about it in
// one round trip to memory: every lane loads its entry of every array, the
// entry wanted is the last whose first work item is not past the wave's, and
// its fields are broadcast into scalar registers. (A search, and then the
// fields it leads to, would be three or four trips one after another, about a
// microsecond of a kernel that lasts four.)
#pragma once

#include "common.h"

namespace prana {

constexpr int kTableSeqs = 64;  // sequences of one launch: the lanes of a wave

// first: the sequences' first work items, ascending.
__device__ __forceinline__ int table_find(const uint32_t* first, uint32_t n_seq, uint32_t item) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t at = __ballot(lane < n_seq && first[lane] <= item);
  return __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(at | 1));
}

__device__ __forceinline__ uint32_t table_pick(uint32_t mine, int seq) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), seq));
}
template <class T>
__device__ __forceinline__ T* table_pick(T* mine, int seq) {
  const uint64_t p = reinterpret_cast<uint64_t>(mine);
  return reinterpret_cast<T*>(static_cast<uint64_t>(table_pick(static_cast<uint32_t>(p >> 32), seq)) << 32 |
                              table_pick(static_cast<uint32_t>(p), seq));
}
// Entry seq of an array of the table.
template <class T>
__device__ __forceinline__ T table_at(const T* array, int seq) {
  return table_pick(array[threadIdx.x & 63], seq);
}

}  // namespace prana
