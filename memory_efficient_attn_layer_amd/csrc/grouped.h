// Host interface of the grouped, paged and tree attention kernels: parameter
// structs and launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mea {

typedef uint16_t bits16;

// Attention of packed sequences, Hq query heads over Hkv key/value heads.
// Tokens outside every sequence (before cu[0], from cu[nseq] on) get zeros.
struct GroupedParams {
  const bits16 *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;  // strides in elements
  const int* cu;                                        // (nseq + 1)
  int nseq, total, Hq, Hkv;
  float scale, sl2e;  // softmax scale; scale * log2(e)
  bits16* o;          // (total, Hq, N)
  // For a backward (bf16): both or neither.
  bits16* o_rest;  // (total, Hq, N): what rounding o to 16 bits left
  float* lse;      // (Hq, total)
  // backward
  const bits16* dO;                                     // (total, Hq, N)
  const float* lse_in;                                  // (Hq, total)
  float* delta;                                         // (Hq, total), from dq for dk and dv
  bits16 *dq, *dk, *dv;                                 // (total, Hq | Hkv, N)
  int parts;    // of the dk/dv sums (dkdv_parts)
  float* sums;  // (parts, 2, total, Hkv, N) where parts > 1
};
int dkdv_parts(int total, int nseq, int Hq, int Hkv, int N);
hipError_t launch_grouped_fwd(const GroupedParams& p, int N, bool fp16, hipStream_t s);
hipError_t launch_grouped_dq(const GroupedParams& p, int N, hipStream_t s);
hipError_t launch_grouped_dkdv(const GroupedParams& p, int N, hipStream_t s);
hipError_t launch_grouped_join(const GroupedParams& p, int N, hipStream_t s);

// A cache of fixed-size pages. Sequence s holds rows 0 .. lengths[s]-1; row r is
// row r % page of page table[s][r / page] of both pools. refs counts the table
// entries that hold a page; a page with none is free.
struct PagedCache {
  bits16 *k, *v;               // (pages, Hkv, page, N)
  int *table, *lengths, *refs, *status;  // (seqs, max_pages), (seqs), (pages), (1)
  int seqs, pages, Hkv, page, lg_page, N, max_pages;
};
// Bits of *status.
constexpr int kNoPages = 1;  // a call found fewer free pages than it needed
constexpr int kNoRows = 2;   // a sequence would pass max_pages

// New rows: token t of sequence s at k + s * seq + t * tok + head * head (uniform,
// n tokens each) or, with cu, at k + t * tok + head * head for t in cu[s] .. cu[s+1]-1.
struct AppendParams {
  PagedCache c;
  const bits16 *k, *v;
  int64_t k_seq, k_tok, k_head, v_seq, v_tok, v_head;
  const int* cu;
  int n, total;
  int* ws;  // append_ws_ints()
};
struct AcceptParams {
  PagedCache c;
  const int *path, *counts;  // (seqs, most), (seqs)
  int n, most;
  int* ws;  // accept_ws_ints()
};
size_t append_ws_ints(int seqs, int pages);
size_t accept_ws_ints(int seqs, int pages, int page, int n);
size_t fork_ws_ints(int seqs, int max_pages);
size_t compact_ws_ints(int pages);
hipError_t launch_paged_append_plan(const AppendParams& p, hipStream_t s);
hipError_t launch_paged_append_rows(const AppendParams& p, hipStream_t s);
hipError_t launch_paged_accept_plan(const AcceptParams& p, hipStream_t s);
hipError_t launch_paged_accept_rows(const AcceptParams& p, hipStream_t s);
hipError_t launch_paged_truncate(const PagedCache& c, const int* lengths, hipStream_t s);
bool paged_fork_small(const PagedCache& c);  // launch_paged_fork takes it; else the two launches
hipError_t launch_paged_fork(const PagedCache& c, const int* parents, hipStream_t s);
hipError_t launch_paged_fork_read(const PagedCache& c, const int* parents, int* ws, hipStream_t s);
hipError_t launch_paged_fork_write(const PagedCache& c, const int* parents, const int* ws, hipStream_t s);
hipError_t launch_paged_compact_plan(const PagedCache& c, int* ws, hipStream_t s);
hipError_t launch_paged_compact_move(const PagedCache& c, const int* ws, hipStream_t s);

// Attention of n new tokens per sequence (the last n rows of each) over a paged cache.
constexpr int kMaxTree = 256;  // new tokens per sequence
struct TreeParams {
  PagedCache c;
  const bits16* q;  // (seqs, n, Hq, N)
  int64_t q_seq, q_tok, q_head;
  const unsigned char* mask;  // (n, n) bytes per sequence, mask_seq apart (0: one for all); null: causal
  int64_t mask_seq;
  int n, Hq, want, least, full, row_groups;  // from want on: of TreeGrid
  float sl2e;
  bits16* o;    // (seqs, n, Hq, N)
  // Null where no sequence can have two chunks: first item and chunks of each
  // sequence, then (items, Hkv, rows) of N + 4 floats (the sums, m, l), rows = n * Hq / Hkv.
  float* part;
};
__host__ __device__ inline size_t tree_head_floats(int seqs) { return (2 * (size_t)seqs + 3) & ~(size_t)3; }
// How a call is cut up. full: the largest chunks of a sequence of all the rows that it
// can have; split: a sequence may have several chunks, whose sums the second launch
// joins.
struct TreeGrid {
  int blocks, row_groups, turn, want, least, full;
  int64_t items;
  bool split;
};
TreeGrid tree_grid(int seqs, int Hkv, int rows, int capacity, int N);
hipError_t launch_tree_attn(const TreeParams& p, bool fp16, hipStream_t s);
hipError_t launch_tree_combine(const TreeParams& p, bool fp16, hipStream_t s);

}  // namespace mea
