// The paged cache's own operators: new rows in, the accepted rows of a drafted
// tree together, pages shared, given back and moved to the front of the pool.
//
// Everything the operators decide (which page is free, which sequence has room)
// is decided on the GPU, so that a decoding loop neither waits for it nor leaves
// a captured graph. A plan is one workgroup: needs per sequence, a scan over
// them, the lowest free pages in order from a scan over the counts, and the
// table's new entries; a second launch moves the rows, bound by HBM. Nothing
// depends on the order of atomics: counts are sums, and who gets which page
// follows from the order of sequences and pages alone.
//
// A page held by more than one sequence is never written: a sequence that writes
// into one gets a page of its own with a copy of the rows it has in it. Pages
// given back by a call are free for the next call, not within it, so no row is
// read that the same call overwrites.
//
// Table entries outside the pool are skipped wherever they are met.
#include "common.cuh"
#include "grouped.h"

namespace mea {

namespace {

constexpr int kPlan = 1024;  // threads of a plan

// Exclusive scan over the workgroup's kPlan threads; *total gets the sum. Two
// barriers; lds holds kPlan / 64 + 1 ints and is free again after the next one.
__device__ __forceinline__ int block_scan(int v, int* lds, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) {
    const int y = lds[w];
    before += w < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before + x - v;
}

__device__ __forceinline__ bool in_pool(const PagedCache& c, int page) { return (unsigned)page < (unsigned)c.pages; }
__device__ __forceinline__ int length_of(const PagedCache& c, int s) {
  return min(max(c.lengths[s], 0), c.max_pages << c.lg_page);
}
__device__ __forceinline__ int pages_of(const PagedCache& c, int rows) { return (rows + c.page - 1) >> c.lg_page; }
// First element of (page, head, row).
__device__ __forceinline__ size_t row_at(const PagedCache& c, int page, int head, int row) {
  return ((((size_t)page * c.Hkv + head) << c.lg_page) + row) * c.N;
}

// Bit e: page at + e is free, for the four pages of a thread.
__device__ __forceinline__ int free_four(const PagedCache& c, int at) {
  int bits = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) bits |= (int)(at + e < c.pages && c.refs[min(at + e, c.pages - 1)] <= 0) << e;
  return bits;
}
// The lowest `need` free pages into list, in order; returns how many there are
// (all threads, after a barrier). first: free_four() of the thread's first four
// pages, which the caller requests before it knows the need.
__device__ __forceinline__ int free_pages(const PagedCache& c, int need, int first, int* list, int* lds) {
  int found = 0;
  for (int p0 = 0; p0 < c.pages && found < need; p0 += 4 * kPlan) {
    const int at = p0 + 4 * threadIdx.x, free = p0 == 0 ? first : free_four(c, at);
    int total, rank = found + block_scan(__popc(free), lds, &total);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is = (free >> e & 1) != 0;
      if (is && rank < need) list[rank] = at + e;
      rank += is;
    }
    found += total;
  }
  __syncthreads();
  return min(found, need);
}

// Workspaces (ints): per sequence [start | copied page | three notes], then the list
// of free pages.
struct AppendWs {
  int *start, *copied, *notes, *list;
};
__host__ __device__ AppendWs append_ws(int* ws, int S) { return AppendWs{ws, ws + S, ws + 2 * S, ws + 5 * S}; }
__host__ __device__ inline int tree_pages(int page, int n) { return (n + page - 1) / page + 1; }
struct AcceptWs {
  int *base, *count, *need, *off, *shared, *old, *list;  // old: (S, J) pages before the call
};
__host__ __device__ AcceptWs accept_ws(int* ws, int S, int J) {
  return AcceptWs{ws, ws + S, ws + 2 * S, ws + 3 * S, ws + 4 * S, ws + 5 * S, ws + 5 * S + (size_t)S * J};
}

__device__ __forceinline__ int new_rows(const AppendParams& p, int s) {
  if (p.cu == nullptr) return p.n;
  const int a = min(max(p.cu[s], 0), p.total);
  return min(max(p.cu[s + 1], a), p.total) - a;
}

// Up to kPlan sequences, what the plan knows of them stays in LDS from the first
// half to the second (9.3 -> 5.4 us at 64 sequences).
template <int FIELDS>
struct PlanNotes {
  int* at[FIELDS];
  __device__ __forceinline__ PlanNotes(int* lds, int* ws, int seqs) {
    const bool fits = seqs <= kPlan;
#pragma unroll
    for (int f = 0; f < FIELDS; ++f) at[f] = fits ? lds + f * kPlan : ws + (size_t)f * seqs;
  }
  __device__ __forceinline__ int& operator()(int f, int s) const { return at[f][s]; }
};

__global__ __launch_bounds__(kPlan) void append_plan_kernel(AppendParams p) {
  __shared__ int lds[kPlan / 64], notes_lds[3 * kPlan];
  const PagedCache& c = p.c;
  const AppendWs w = append_ws(p.ws, c.seqs);
  enum { OLD, NEED, OFF };  // rows before; pages needed (-1: no room for the rows); first of them
  const PlanNotes<3> note(notes_lds, w.notes, c.seqs);
  const int tid = threadIdx.x;
  const int first_free = free_four(c, 4 * tid);
  int total = 0;
  for (int s0 = 0; s0 < c.seqs; s0 += kPlan) {
    const int s = s0 + tid;
    int need = 0, copied = -1, old = 0;
    if (s < c.seqs) {
      const int more = new_rows(p, s);
      old = length_of(c, s);
      if (more > 0 && more <= (c.max_pages << c.lg_page) - old) {
        need = pages_of(c, old + more) - pages_of(c, old);
        if ((old & (c.page - 1)) != 0) {
          const int tail = c.table[(size_t)s * c.max_pages + (old >> c.lg_page)];
          if (in_pool(c, tail) && c.refs[tail] > 1) {
            copied = tail;
            ++need;
          }
        }
      } else if (more > 0) {
        need = -1;
      }
    }
    int sum;
    const int off = total + block_scan(max(need, 0), lds, &sum);
    total += sum;
    if (s < c.seqs) {
      w.copied[s] = copied;
      note(OLD, s) = old;
      note(NEED, s) = need;
      note(OFF, s) = off;
    }
  }
  const int found = free_pages(c, total, first_free, w.list, lds);
  // Who is served is settled; now the sequences' own entries.
  for (int s = tid; s < c.seqs; s += kPlan) {
    const int need = note(NEED, s), old = note(OLD, s), copied = w.copied[s];
    const bool ok = need >= 0 && (need == 0 || note(OFF, s) + need <= found);
    w.start[s] = ok ? old : -1;
    if (!ok) {
      w.copied[s] = -1;
      atomicOr(c.status, need < 0 ? kNoRows : kNoPages);
      note(NEED, s) = 0;
    } else {
      const int more = new_rows(p, s);
      if (copied >= 0) atomicSub(&c.refs[copied], 1);
      if (more > 0) c.lengths[s] = old + more;
      // The first entry that is set: the copied page's, or the one behind the last.
      note(OLD, s) = pages_of(c, old) - (copied >= 0 ? 1 : 0);
    }
  }
  __syncthreads();
  // Pages: a wave per sequence where there are many, a thread where there are one or two.
  const int lane = tid & 63;
  if (total <= 4 * c.seqs) {
    for (int s = tid; s < c.seqs; s += kPlan)
      for (int j = 0; j < note(NEED, s); ++j) {
        const int page = w.list[note(OFF, s) + j];
        c.table[(size_t)s * c.max_pages + note(OLD, s) + j] = page;
        c.refs[page] = 1;
      }
    return;
  }
  for (int s = tid >> 6; s < c.seqs; s += kPlan / 64)
    for (int j = lane; j < note(NEED, s); j += 64) {
      const int page = w.list[note(OFF, s) + j];
      c.table[(size_t)s * c.max_pages + note(OLD, s) + j] = page;
      c.refs[page] = 1;
    }
}

// Workgroups [0, row_wgs): 16-byte chunks of the new rows, chunk fastest. The
// rest: one per (sequence, head), the rows of a copied last page.
__global__ __launch_bounds__(256) void append_rows_kernel(AppendParams p, int row_wgs) {
  const PagedCache& c = p.c;
  const AppendWs w = append_ws(p.ws, c.seqs);
  const int CH = c.N / 8;
  if ((int)blockIdx.x < row_wgs) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int per = c.Hkv * CH;
    const int t = (int)(id / per), r = (int)(id - (int64_t)t * per), head = r / CH, ch = r - head * CH;
    const int rows = p.cu == nullptr ? c.seqs * p.n : p.total;
    if (t >= rows) return;
    int s, i;
    int64_t src_k, src_v;
    if (p.cu == nullptr) {
      s = t / p.n;
      i = t - s * p.n;
      src_k = s * p.k_seq + i * p.k_tok;
      src_v = s * p.v_seq + i * p.v_tok;
    } else {
      // The last sequence that begins at or before t.
      int lo = 0, hi = c.seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (p.cu[mid] <= t ? lo : hi) = mid;
      }
      s = lo;
      i = t - max(p.cu[s], 0);
      if (i < 0 || i >= new_rows(p, s)) return;  // a token of no sequence
      src_k = t * p.k_tok;
      src_v = t * p.v_tok;
    }
    const int start = w.start[s];
    if (start < 0) return;
    const int row = start + i, page = c.table[(size_t)s * c.max_pages + (row >> c.lg_page)];
    if (!in_pool(c, page)) return;
    const size_t at = row_at(c, page, head, row & (c.page - 1)) + ch * 8;
    const u32x4 kv = ld16(p.k + src_k + head * p.k_head + ch * 8), vv = ld16(p.v + src_v + head * p.v_head + ch * 8);
    st16(c.k + at, kv);
    st16(c.v + at, vv);
    return;
  }
  const int e = blockIdx.x - row_wgs, s = e / c.Hkv, head = e - s * c.Hkv;
  const int from = w.copied[s];
  if (from < 0) return;
  const int start = w.start[s], to = c.table[(size_t)s * c.max_pages + (start >> c.lg_page)];
  if (!in_pool(c, to)) return;
  const size_t a = row_at(c, from, head, 0), b = row_at(c, to, head, 0);
  for (int id = threadIdx.x; id < (start & (c.page - 1)) * CH; id += 256) {
    const u32x4 kv = ld16(c.k + a + id * 8), vv = ld16(c.v + a + id * 8);
    st16(c.k + b + id * 8, kv);
    st16(c.v + b + id * 8, vv);
  }
}

__global__ __launch_bounds__(kPlan) void accept_plan_kernel(AcceptParams p) {
  __shared__ int lds[kPlan / 64];
  const PagedCache& c = p.c;
  const int J = tree_pages(c.page, p.n), tid = threadIdx.x;  // J <= 17
  const AcceptWs w = accept_ws(p.ws, c.seqs, J);
  const int first_free = free_four(c, 4 * tid);
  int total = 0;
  for (int s0 = 0; s0 < c.seqs; s0 += kPlan) {
    const int s = s0 + tid;
    int need = 0;
    if (s < c.seqs) {
      const int len = length_of(c, s), base = max(len - p.n, 0);
      const int count = min(max(p.counts[s], 0), min(p.most, len - base));
      const int p0 = base >> c.lg_page, pe = count > 0 ? pages_of(c, base + count) : p0;
      int shared = 0;
      for (int j = 0; p0 + j < pe; ++j) {
        const int page = c.table[(size_t)s * c.max_pages + p0 + j];
        if (in_pool(c, page) && c.refs[page] > 1) {
          shared |= 1 << j;
          ++need;
        }
      }
      w.base[s] = base;
      w.count[s] = count;
      w.shared[s] = shared;
      w.need[s] = need;
    }
    int sum;
    const int off = total + block_scan(need, lds, &sum);
    total += sum;
    if (s < c.seqs) w.off[s] = off;
  }
  const int found = free_pages(c, total, first_free, w.list, lds);
  const int lane = tid & 63;
  for (int s = tid >> 6; s < c.seqs; s += kPlan / 64) {
    const int need = w.need[s], off = w.off[s], base = w.base[s], count = w.count[s], shared = w.shared[s];
    const int len = length_of(c, s);
    if (need > 0 && off + need > found) {
      if (lane == 0) {
        w.count[s] = 0;
        w.shared[s] = 0;
        atomicOr(c.status, kNoPages);
      }
      continue;
    }
    const int p0 = base >> c.lg_page, held = pages_of(c, len), keep = pages_of(c, base + count);
    if (lane < J) {
      const int slot = p0 + lane;
      int* entry = c.table + (size_t)s * c.max_pages + slot;
      const int page = slot < held ? *entry : -1;
      w.old[(size_t)s * J + lane] = page;
      if ((shared >> lane & 1) != 0) {
        const int mine = w.list[off + __popc(shared & ((1 << lane) - 1))];
        *entry = mine;
        c.refs[mine] = 1;
        atomicSub(&c.refs[page], 1);
      } else if (slot >= keep && slot < held) {
        *entry = -1;
        if (in_pool(c, page)) atomicSub(&c.refs[page], 1);
      }
    }
    if (lane == 0) {
      w.need[s] = len - base;  // rows of the tree
      c.lengths[s] = base + count;
    }
  }
}

// One workgroup per (sequence, head, pool and 64-column slab): the accepted rows
// are all read before the first is written, so the path may name any rows in any
// order; kMaxTree rows of 8 chunks are 8 registers of 16 bytes a thread.
__global__ __launch_bounds__(256) void accept_rows_kernel(AcceptParams p) {
  const PagedCache& c = p.c;
  const int J = tree_pages(c.page, p.n), s = blockIdx.x, head = blockIdx.y;
  const AcceptWs w = accept_ws(p.ws, c.seqs, J);
  const int count = w.count[s], base = w.base[s], shared = w.shared[s], rows = w.need[s];
  if (count == 0) return;
  bits16* pool = blockIdx.z & 1 ? c.v : c.k;
  const int CH = min(c.N / 8, 8), c0 = (blockIdx.z >> 1) * 64;
  const int p0 = base >> c.lg_page, mask = c.page - 1;
  const int* old = w.old + (size_t)s * J;
  const int* now = c.table + (size_t)s * c.max_pages + p0;
  const int last = base - (p0 << c.lg_page);  // first row of the tree in its first page
  constexpr int R = kMaxTree * 8 / 256;
  u32x4 val[R];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int id = threadIdx.x + 256 * u, i = id / CH, ch = id - i * CH;
    if (i >= count) continue;
    const int row = last + min(max(p.path[(size_t)s * p.most + i], 0), rows - 1);
    const int page = old[row >> c.lg_page];
    if (in_pool(c, page)) val[u] = ld16(pool + row_at(c, page, head, row & mask) + c0 + ch * 8);
  }
  if ((shared & 1) != 0 && in_pool(c, now[0])) {  // the rows in front of the tree
    const size_t a = row_at(c, old[0], head, 0) + c0, b = row_at(c, now[0], head, 0) + c0;
    for (int id = threadIdx.x; id < last * CH; id += 256) {
      const size_t at = (size_t)(id / CH) * c.N + id % CH * 8;
      st16(pool + b + at, ld16(pool + a + at));
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int id = threadIdx.x + 256 * u, i = id / CH, ch = id - i * CH;
    if (i >= count) continue;
    const int src = last + min(max(p.path[(size_t)s * p.most + i], 0), rows - 1), row = last + i;
    const int from = old[src >> c.lg_page], page = now[row >> c.lg_page];
    if (in_pool(c, page) && in_pool(c, from)) st16(pool + row_at(c, page, head, row & mask) + c0 + ch * 8, val[u]);
  }
}

__global__ __launch_bounds__(64) void truncate_kernel(PagedCache c, const int* lengths) {
  const int s = blockIdx.x, old = length_of(c, s), len = min(max(lengths[s], 0), old);
  for (int j = pages_of(c, len) + threadIdx.x; j < pages_of(c, old); j += 64) {
    int* entry = c.table + (size_t)s * c.max_pages + j;
    if (in_pool(c, *entry)) atomicSub(&c.refs[*entry], 1);
    *entry = -1;
  }
  if (threadIdx.x == 0) c.lengths[s] = len;
}

// Fork, first half: sequence s's new entries (its parent's) into the workspace
// and the counts; second half: the entries into the table. (In one launch a row
// could be overwritten before its children have read it.)
__global__ __launch_bounds__(256) void fork_read_kernel(PagedCache c, const int* parents, int* ws) {
  const int s = blockIdx.x, from = parents[s];
  if (from == s) return;
  const bool live = (unsigned)from < (unsigned)c.seqs;
  const int len = live ? length_of(c, from) : 0, held = pages_of(c, len), was = pages_of(c, length_of(c, s));
  int* row = ws + c.seqs + (size_t)s * c.max_pages;
  for (int j = threadIdx.x; j < max(held, was); j += 256) {
    if (j < held) {
      const int page = c.table[(size_t)from * c.max_pages + j];
      row[j] = page;
      if (in_pool(c, page)) atomicAdd(&c.refs[page], 1);
    }
    if (j < was) {
      const int page = c.table[(size_t)s * c.max_pages + j];
      if (in_pool(c, page)) atomicSub(&c.refs[page], 1);
    }
  }
  if (threadIdx.x == 0) ws[s] = len;
}
__global__ __launch_bounds__(256) void fork_write_kernel(PagedCache c, const int* parents, const int* ws) {
  const int s = blockIdx.x;
  if (parents[s] == s) return;
  const int len = ws[s], held = pages_of(c, len), was = pages_of(c, length_of(c, s));
  const int* row = ws + c.seqs + (size_t)s * c.max_pages;
  __syncthreads();  // the old length is read
  for (int j = threadIdx.x; j < max(held, was); j += 256)
    c.table[(size_t)s * c.max_pages + j] = j < held ? row[j] : -1;
  if (threadIdx.x == 0) c.lengths[s] = len;
}

// Both halves in one workgroup, where the table fits its LDS (two launches: 3.5 + 2.6
// us at 64 sequences of 65 entries).
constexpr int kForkEntries = 12288;
__global__ __launch_bounds__(kPlan) void fork_small_kernel(PagedCache c, const int* parents) {
  __shared__ int rows[kForkEntries], len_s[kPlan], from_s[kPlan], pages_s[kPlan];
  const int tid = threadIdx.x, n = c.seqs * c.max_pages;
  int len = 0;
  if (tid < c.seqs) {
    const int from = parents[tid];
    from_s[tid] = (unsigned)from < (unsigned)c.seqs ? from : -1;
    len_s[tid] = len = length_of(c, tid);
    pages_s[tid] = pages_of(c, len);
  }
  for (int i = tid; i < n; i += kPlan) rows[i] = c.table[i];
  __syncthreads();
  for (int i = tid; i < n; i += kPlan) {
    const int s = i / c.max_pages, j = i - s * c.max_pages, from = from_s[s];
    if (from == s) continue;
    const int was = j < pages_s[s] ? rows[i] : -1;
    const int now = from >= 0 && j < pages_s[from] ? rows[from * c.max_pages + j] : -1;
    if (was == now) continue;  // the same page stays: nothing to count
    if (in_pool(c, now)) atomicAdd(&c.refs[now], 1);
    if (in_pool(c, was)) atomicSub(&c.refs[was], 1);
    c.table[i] = now;
  }
  if (tid < c.seqs && from_s[tid] != tid) c.lengths[tid] = from_s[tid] >= 0 ? len_s[from_s[tid]] : 0;
}

// Workspace: [count of moves][page -> new page][sources][targets]. Four pages a
// thread and pass (one page: 11.3 us, four: 6.5, of 3100 pages).
__global__ __launch_bounds__(kPlan) void compact_plan_kernel(PagedCache c, int* ws) {
  __shared__ int lds[kPlan / 64];
  int *map = ws + 1, *src = map + c.pages, *dst = src + c.pages;
  const int first = free_four(c, 4 * threadIdx.x);
  auto free_at = [&](int at) { return at < 4 * kPlan ? first : free_four(c, at); };
  auto real = [&](int at) { return at >= c.pages ? 0 : at + 4 <= c.pages ? 15 : (1 << (c.pages - at)) - 1; };
  int live = 0;
  for (int p0 = 0; p0 < c.pages; p0 += 4 * kPlan) {
    int total;
    const int at = p0 + 4 * threadIdx.x;
    block_scan(__popc(real(at) & ~free_at(at)), lds, &total);
    live += total;
  }
  int n_src = 0, n_dst = 0;
  for (int p0 = 0; p0 < c.pages; p0 += 4 * kPlan) {
    const int at = p0 + 4 * threadIdx.x, free = free_at(at), used = real(at) & ~free;
    const int low = at >= live ? 0 : at + 4 <= live ? 15 : (1 << (live - at)) - 1;  // pages below live
    const int moves = used & ~low, holes = free & low;
    int total;
    // Holes lie before the moving pages, but both may share a pass: a half each, 4 * kPlan at most.
    const int packed = block_scan(__popc(moves) | __popc(holes) << 16, lds, &total);
    int to_src = n_src + (packed & 0xFFFF), to_dst = n_dst + (packed >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((moves >> e & 1) != 0) src[to_src++] = at + e;
      if ((holes >> e & 1) != 0) dst[to_dst++] = at + e;
      if (at + e < c.pages) map[at + e] = at + e;
    }
    n_src += total & 0xFFFF;
    n_dst += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_src; i += kPlan) map[src[i]] = dst[i];
  if (threadIdx.x == 0) ws[0] = n_src;
}

__global__ __launch_bounds__(256) void compact_move_kernel(PagedCache c, const int* ws) {
  const int *map = ws + 1, *src = map + c.pages, *dst = src + c.pages;
  const int n = ws[0];
  if (n == 0) return;
  constexpr int PART = 2048;  // 16-byte chunks a workgroup moves at a time
  const int chunks = (c.Hkv << c.lg_page) * (c.N / 8), parts = (chunks + PART - 1) / PART;
  for (int64_t i = blockIdx.x; i < (int64_t)n * parts; i += gridDim.x) {
    const int m = (int)(i / parts), part = (int)(i - (int64_t)m * parts);
    const size_t a = (size_t)src[m] * chunks * 8, b = (size_t)dst[m] * chunks * 8;
    const int end = min(chunks, (part + 1) * PART);
    for (int id = part * PART + threadIdx.x; id < end; id += 256) {
      const u32x4 kv = ld16(c.k + a + (size_t)id * 8), vv = ld16(c.v + a + (size_t)id * 8);
      st16(c.k + b + (size_t)id * 8, kv);
      st16(c.v + b + (size_t)id * 8, vv);
    }
    if (part == 0 && threadIdx.x == 0) {
      c.refs[dst[m]] = c.refs[src[m]];
      c.refs[src[m]] = 0;
    }
  }
  const int64_t entries = (int64_t)c.seqs * c.max_pages;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
    const int page = c.table[i];
    if (in_pool(c, page) && map[page] != page) c.table[i] = map[page];
  }
}

}  // namespace

size_t append_ws_ints(int seqs, int pages) { return 5 * (size_t)seqs + pages; }
size_t accept_ws_ints(int seqs, int pages, int page, int n) {
  return (size_t)seqs * (5 + tree_pages(page, n)) + pages;
}
size_t fork_ws_ints(int seqs, int max_pages) { return (size_t)seqs * (1 + (size_t)max_pages); }
size_t compact_ws_ints(int pages) { return 1 + 3 * (size_t)pages; }

hipError_t launch_paged_append_plan(const AppendParams& p, hipStream_t s) {
  hipLaunchKernelGGL(append_plan_kernel, dim3(1), dim3(kPlan), 0, s, p);
  return hipGetLastError();
}
hipError_t launch_paged_append_rows(const AppendParams& p, hipStream_t s) {
  const int64_t rows = p.cu == nullptr ? (int64_t)p.c.seqs * p.n : p.total;
  const int row_wgs = (int)((rows * p.c.Hkv * (p.c.N / 8) + 255) / 256);
  hipLaunchKernelGGL(append_rows_kernel, dim3(row_wgs + p.c.seqs * p.c.Hkv), dim3(256), 0, s, p, row_wgs);
  return hipGetLastError();
}
hipError_t launch_paged_accept_plan(const AcceptParams& p, hipStream_t s) {
  hipLaunchKernelGGL(accept_plan_kernel, dim3(1), dim3(kPlan), 0, s, p);
  return hipGetLastError();
}
hipError_t launch_paged_accept_rows(const AcceptParams& p, hipStream_t s) {
  const int slabs = (p.c.N + 63) / 64;
  hipLaunchKernelGGL(accept_rows_kernel, dim3(p.c.seqs, p.c.Hkv, 2 * slabs), dim3(256), 0, s, p);
  return hipGetLastError();
}
hipError_t launch_paged_truncate(const PagedCache& c, const int* lengths, hipStream_t s) {
  hipLaunchKernelGGL(truncate_kernel, dim3(c.seqs), dim3(64), 0, s, c, lengths);
  return hipGetLastError();
}
bool paged_fork_small(const PagedCache& c) {
  return c.seqs <= kPlan && (int64_t)c.seqs * c.max_pages <= kForkEntries;
}
hipError_t launch_paged_fork(const PagedCache& c, const int* parents, hipStream_t s) {
  hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kPlan), 0, s, c, parents);
  return hipGetLastError();
}
hipError_t launch_paged_fork_read(const PagedCache& c, const int* parents, int* ws, hipStream_t s) {
  hipLaunchKernelGGL(fork_read_kernel, dim3(c.seqs), dim3(256), 0, s, c, parents, ws);
  return hipGetLastError();
}
hipError_t launch_paged_fork_write(const PagedCache& c, const int* parents, const int* ws, hipStream_t s) {
  hipLaunchKernelGGL(fork_write_kernel, dim3(c.seqs), dim3(256), 0, s, c, parents, ws);
  return hipGetLastError();
}
hipError_t launch_paged_compact_plan(const PagedCache& c, int* ws, hipStream_t s) {
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlan), 0, s, c, ws);
  return hipGetLastError();
}
hipError_t launch_paged_compact_move(const PagedCache& c, const int* ws, hipStream_t s) {
  hipLaunchKernelGGL(compact_move_kernel, dim3(2048), dim3(256), 0, s, c, ws);
  return hipGetLastError();
}

}  // namespace mea
