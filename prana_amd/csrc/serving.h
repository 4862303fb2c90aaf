// Packed prompts, 8-bit K/V caches and trees of drafted tokens: the argument
// checks, the plans and the launches behind the serving entry points of
// include/prana_hip.h.
//
// The sequences' sizes and cache pointers travel to the kernels by value (a
// few KB of kernel arguments), so a call neither uploads nor allocates, and a
// captured launch holds everything it needs. Batches of more sequences than
// one launch holds take several launches.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/prana_hip.h"

namespace prana {

// ------------------------------------------------------------ checks (host only, no device call)
int check_heads(const char* what, size_t n_heads, size_t n_kv_heads, size_t head_dim);
int check_attention_packed(const void* q, const uint16_t* k, const uint16_t* v, int type, const size_t* seq_lens,
                           size_t n_seq, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t ld_q,
                           size_t ld_kv, size_t ld_out, const void* out);
// The caches and row ranges of prana_kv_write_q8 / prana_kv_read_q8; src is
// the packed side (k and v, elements of `size` bytes, row stride ld).
int check_kv_q8(const char* what, const prana_kv* kv, const size_t* first_rows, const size_t* n_rows, size_t n_seq,
                size_t n_kv_heads, size_t head_dim, const void* k, const void* v, size_t ld, size_t size);
int check_attention_tree(const float* q, int kv_type, const prana_kv* kv, const size_t* past, const size_t* n_tree,
                         size_t n_seq, const uint64_t* mask, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                         const float* out, const void* workspace, size_t workspace_bytes);
// The sizes alone (what the workspace depends on).
int check_tree_sizes(const size_t* past, const size_t* n_tree, size_t n_seq, size_t n_heads, size_t n_kv_heads,
                     size_t head_dim);

constexpr size_t kMaxTree = 64;  // drafted tokens of a sequence: the bits of a mask word

// ------------------------------------------------------------ packed_attention.hip
// Lanes of the launch that one sequence needs at least: they are to fit 32 bits.
size_t packed_lanes(size_t len, size_t n_heads, size_t n_kv_heads, size_t head_dim);
int launch_attention_packed(const void* q, const uint16_t* k, const uint16_t* v, bool half, const size_t* seq_lens,
                            size_t n_seq, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t ld_q,
                            size_t ld_kv, size_t ld_out, void* out, hipStream_t s);

// ------------------------------------------------------------ kv_q8.hip
int launch_kv_write_q8(const float* k, const float* v, size_t ld, const prana_kv* kv, const size_t* first_rows,
                       const size_t* n_rows, size_t n_seq, size_t n_kv_heads, size_t head_dim, hipStream_t s);
int launch_kv_read_q8(const prana_kv* kv, const size_t* first_rows, const size_t* n_rows, size_t n_seq,
                      size_t n_kv_heads, size_t head_dim, bool half, void* k, void* v, size_t ld, hipStream_t s);

// ------------------------------------------------------------ tree_attention.hip
// Floats of workspace for a call with these sizes, or smaller ones.
size_t attention_tree_floats(const size_t* past, const size_t* n_tree, size_t n_seq, size_t n_heads,
                             size_t n_kv_heads, size_t head_dim);
int launch_attention_tree(const float* q, bool q8, const prana_kv* kv, const size_t* past, const size_t* n_tree,
                          size_t n_seq, const uint64_t* mask, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                          float* out, float* workspace, size_t workspace_floats, hipStream_t s);

}  // namespace prana
