// Causal attention of packed sequences with grouped heads on gfx950 MFMA:
// forward and backward for q (total, Hq, N), k and v (total, Hkv, N), query
// head h reading key/value head h / G, G = Hq / Hkv.
//
//   s_ij = scale q_i . k_j  (j <= i, same sequence)    p_ij = exp(s_ij - lse_i)
//   o_i = sum_j p_ij v_j                               lse_i = log sum_j exp(s_ij)
//   delta_i = dO_i . o_i                               dp_ij = dO_i . v_j
//   ds_ij = p_ij (dp_ij - delta_i)                     dq_i = scale sum_j ds_ij k_j
//   dk_j = scale sum_{heads of the group, i >= j} ds_ij q_i     dv_j = sum p_ij dO_i
//
// The products run on v_mfma_f32_32x32x16 in the operand forms of the block's
// attention kernels (attn_fwd.hip, attn_bwd.hip): tiles of 32 or 64 rows
// through swizzled LDS, the weights fed back as an operand straight from the
// accumulator, sequence-major operands read with the transposing LDS load. The
// weights and ds are rounded to the inputs' 16 bits for their products; every
// sum and statistic is fp32.
//
// What differs: rows are token-major with strides of their own; nothing bounds
// the logits, so the softmax keeps a running maximum; and the four waves of a
// workgroup take `hw` query heads of one group (4, 2 or 1, as G allows) times
// 4 / hw blocks of 32 tokens, so a group's heads share the K/V tiles they load
// and a workgroup of four heads ends at its own 32 tokens' diagonal instead of
// 128 tokens'.
//
// Work list: no host knows the lengths. The boundaries 0, cu[0], ..,
// cu[nseq], total cut the tokens into nseq + 2 segments (the first and the last
// hold no sequence; their outputs are zeros). The blocks of up to 64 segments are taken
// longest first: each lane of a wave holds one segment, and a search over the length
// finds the block. (Segment after segment: 276 us for 268 at 24 sequences of 1100 on
// average, 8 / 4 heads of 64, forward and backward; 1743 for 1714 at two of 8192, 16 / 4
// heads of 128.) Of more segments, segment i owns the virtual blocks from
// b_i / BT + i on (BT tokens a block), which leaves room for ceil(len / BT) of
// them, and a workgroup counts the starts at or below its block, 64 at a time.
#include <type_traits>

#include "elem.cuh"
#include "grouped.h"

namespace mea {

namespace {

struct Segment {
  int start, len, blk;  // first token, tokens, block inside the segment
  bool live;            // holds a sequence (the others get zeros)
};

// Virtual blocks of BT tokens.
__host__ __device__ inline int virtual_blocks(int total, int nseq, int BT) { return total / BT + nseq + 2; }

// The v-th block of the work list. LAST: a segment's last block is its longest (a
// block of queries), else its first (of keys).
template <bool LAST>
__device__ __forceinline__ Segment find_segment(const int* cu, int nseq, int total, int BT, int v) {
  const int lane = threadIdx.x & 63;
  // Boundary i: 0, cu[0] .. cu[nseq], offsets clamped to [0, total].
  auto bound = [&](int i) { return i == 0 ? 0 : i == nseq + 2 ? total : min(max(cu[i - 1], 0), total); };
  Segment s;
  if (nseq + 2 <= 64) {
    const int i = min(lane, nseq + 1), start = bound(i), len = lane < nseq + 2 ? max(bound(i + 1) - start, 0) : 0;
    const int blocks = (len + BT - 1) / BT;
    // A block whose rows meet r blocks of the other side is one of length r; every
    // segment has one of each length up to its own. f(r): blocks of length r or more.
    auto f = [&](int r) { return __builtin_amdgcn_readlane(wave_scan(max(blocks - r + 1, 0)), 63); };
    int r = 1, hi = total / BT + 2, longer = 0;  // f(r) > v >= f(hi) = longer
    if (f(r) <= v) {
      s.start = s.len = s.blk = 0;
      s.live = false;
      return s;
    }
    while (hi - r > 1) {
      const int mid = (r + hi) >> 1, n = f(mid);
      (n > v ? r : hi) = mid;
      if (n <= v) longer = n;
    }
    const unsigned long long has = __ballot(blocks >= r);  // one block each; the (v - longer)-th of them
    const unsigned long long me = __ballot(blocks >= r && __popcll(has & ((1ull << lane) - 1)) == v - longer);
    const int l = __ffsll(me) - 1;
    s.start = __builtin_amdgcn_readlane(start, l);
    s.len = __builtin_amdgcn_readlane(len, l);
    s.blk = LAST ? r - 1 : __builtin_amdgcn_readlane(blocks, l) - r;
    s.live = l > 0 && l <= nseq;
    return s;
  }
  if (LAST) v = virtual_blocks(total, nseq, BT) - 1 - v;
  int n = 0;
  for (int i0 = 0; i0 < nseq + 2; i0 += 64) {
    const int i = i0 + lane;
    n += __popcll(__ballot(i < nseq + 2 && bound(min(i, nseq + 1)) / BT + i <= v));
  }
  const int i = __builtin_amdgcn_readfirstlane(max(n - 1, 0));
  s.start = __builtin_amdgcn_readfirstlane(bound(i));
  s.len = max(__builtin_amdgcn_readfirstlane(bound(i + 1)) - s.start, 0);
  s.blk = v - s.start / BT - i;
  if (s.blk < 0) s.len = s.blk = 0;  // (offsets that decrease: nothing to do)
  s.live = i > 0 && i <= nseq;
  return s;
}

// Key head and first query head of head group hg (hw heads each): key heads
// run fastest, so that consecutive workgroups, which go to the XCDs in turn,
// keep to few key heads per XCD.
struct HeadGroup {
  int kv, q0;
};
__device__ __forceinline__ HeadGroup head_group(int hg, int Hkv, int G, int hw) {
  const int kv = hg % Hkv;
  return HeadGroup{kv, kv * G + hg / Hkv * hw};
}

// Zeros in rows t0 .. t1-1 of `heads` heads from h0 on of an output (total, H, N).
template <int N>
__device__ __forceinline__ void zero_rows(bits16* out, int t0, int t1, int h0, int heads, int H) {
  constexpr int CH = N / 8;
  const int per = heads * CH;
  for (int id = threadIdx.x; id < (t1 - t0) * per; id += blockDim.x) {
    const int t = t0 + id / per, r = id % per;
    st16(out + ((size_t)t * H + h0) * N + r * 8, u32x4{0u, 0u, 0u, 0u});
  }
}

__device__ __forceinline__ int heads_per_wg(int G) { return G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1; }

// Tile loads: lane L of load u fills 16-byte slot L of row block u * 4 + wave of
// a tile of ROWS x N, chunks swizzled. A whole tile comes from a uniform base
// and a lane-constant offset; one that runs past the last row `end` clamps to it.
template <int N, int ROWS>
struct TileLoad {
  static constexpr int CH = N / 8, LOADS = ROWS * CH / 256;
  static_assert(LOADS >= 1, "a tile holds 256 chunks at least");
  int row[LOADS];
  uint32_t col[LOADS];  // bytes

  __device__ __forceinline__ void init(int wave, int lane) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int slot = (u * 4 + wave) * 64 + lane;
      row[u] = slot / CH;
      col[u] = (uint32_t)((slot % CH) ^ chunk_swz<CH>(row[u])) * 16u;
    }
  }
  // Rows j0 .. of base (row stride in elements) into the LDS address lds.
  __device__ __forceinline__ void issue(const bits16* base, int64_t stride, int j0, int end, uint32_t lds, int wave) const {
    const bits16* b = base + (size_t)j0 * stride;
    const uint32_t sb = (uint32_t)stride * 2u;
    const int last = end - 1 - j0;
#pragma unroll
    for (int u = 0; u < LOADS; ++u)
      g2lds16_s(b, (uint32_t)min(row[u], last) * sb + col[u], lds + (uint32_t)(u * 4 + wave) * 1024u);
  }
};

// ---------------------------------------------------------------------------
// Forward. Wave w: query head q0 + w % hw, 32 tokens from (w / hw) * 32 of the
// block on; S^T = K Q^T and O^T += V^T P^T, the query on the lane.
//
// Softmax: the running maximum is not followed score by score. A step first
// takes the weights against the maximum m that is in force, and only where their
// sum passes E::kMaxWeight (or is no number: the first step, m = -inf) finds the
// step's own maximum, rescales and takes them again. The quotient is the same;
// bf16 weights and fp32 sums have the range for it, and the exchange with the
// other half of the wave leaves every other step.
//
// SAVE (a backward follows): lse is taken from the sum of the unrounded weights,
// which the backward's p = exp(s - lse) need, and what O loses in its rounding is
// kept in a second tensor of 16 bits: delta = dO . O cancels against dO . v, and
// from the rounded O its error reaches dq and dk at up to twice their own
// rounding (T = 512, N = 64, logits of standard deviation 4: dq 4.8e-3 off its
// norm, with the rest 2.8e-3, with delta exact 2.5e-3).
// ---------------------------------------------------------------------------
template <class E, int N, bool SAVE>
__global__ __launch_bounds__(256, N <= 64 ? 3 : N == 128 ? 2 : 1) void grouped_fwd_kernel(GroupedParams p) {
  constexpr int BKV = 64;  // keys per LDS tile
  constexpr int CH = N / 8, KS = N / 16, DB = N / 32;
  constexpr int TILE = BKV * N;
  constexpr int OP = N + 8;  // output staging pitch
  constexpr int SMEM = 4 * TILE > 4 * 32 * OP ? 4 * TILE : 4 * 32 * OP;
  __shared__ __attribute__((aligned(16))) bits16 smem[SMEM];  // [stage][K | V], then output staging

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.Hq / p.Hkv, hw = heads_per_wg(G), BT = 128 / hw, NH = p.Hq / hw;
  const HeadGroup hg = head_group(blockIdx.x % NH, p.Hkv, G, hw);
  const Segment sg = find_segment<true>(p.cu, p.nseq, p.total, BT, blockIdx.x / NH);
  const int T = sg.len, b0 = sg.blk * BT;
  if (b0 >= T) return;  // uniform, before any barrier
  if (!sg.live) {
    zero_rows<N>(p.o, sg.start + b0, sg.start + min(b0 + BT, T), hg.q0, hw, p.Hq);
    if (SAVE) zero_rows<N>(p.o_rest, sg.start + b0, sg.start + min(b0 + BT, T), hg.q0, hw, p.Hq);
    return;
  }
  const int c = lane & 31, h = lane >> 5;
  const int head = hg.q0 + wave % hw;
  const int q0w = b0 + wave / hw * 32;
  const int kv_end = min(T, b0 + BT);
  const bits16* kg = p.k + (size_t)sg.start * p.k_tok + (size_t)hg.kv * p.k_head;
  const bits16* vg = p.v + (size_t)sg.start * p.v_tok + (size_t)hg.kv * p.v_head;

  u32x4 qf[KS];  // Q^T fragments (B operand): query q0w + c, d = 16 ks + 8 h
  {
    const bits16* qr = p.q + (size_t)(sg.start + min(q0w + c, T - 1)) * p.q_tok + (size_t)head * p.q_head + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = ld16(qr + 16 * ks);
  }
  TileLoad<N, BKV> tl;
  tl.init(wave, lane);
  const uint32_t smem_b = lds_addr(smem);
  auto issue_tile = [&](int j0, int stage) {
    const uint32_t at = smem_b + (uint32_t)(stage * 2 * TILE) * 2u;
    tl.issue(kg, p.k_tok, j0, T, at, wave);
    tl.issue(vg, p.v_tok, j0, T, at + TILE * 2u, wave);
  };

  float m_i = -INFINITY, l_i = 0.f, l_exact = 0.f;  // sums of weights over this lane's half of the keys
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();

  const int g16 = lane >> 4, i16 = lane & 15;
  const int tr_row = 4 * h + (i16 >> 2), tr_col = 16 * (g16 & 1) + 4 * (i16 & 3);
  int koff[KS], voff[2][DB];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = swz_off<CH>(c, 16 * ks + 8 * h);
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int db = 0; db < DB; ++db) voff[x][db] = swz_off<CH>(tr_row + 8 * x, 32 * db + tr_col);

  // One 32-key step. MASK: it touches the causal diagonal or the sequence's end;
  // infinities and NaN of V are left out there (a weight of 0 would make NaN of
  // them in the rows that do not see their key) and added at the end.
  bool hidden = false;
  auto step = [&](const bits16* kt, const bits16* vt, int kb0, auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    auto scores = [&] {
      f32x16 s = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = E::mma(*reinterpret_cast<const u32x4*>(kt + koff[ks]), qf[ks], s);
      if (MASK) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = kb0 + 8 * (i >> 2) + 4 * h + (i & 3);
          if (key > q0w + c || key >= T) s[i] = -INFINITY;
        }
      }
      return s;
    };
    u32x4 pf[2];
    float ls;  // sum of the step's weights
    auto weigh = [&](f32x16& s) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fast_exp2(__builtin_fmaf(s[i], p.sl2e, -m_i));
#pragma unroll
      for (int kst = 0; kst < 2; ++kst)
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[kst][e] = E::pack(s[8 * kst + 2 * e], s[8 * kst + 2 * e + 1]);
      ls = E::add_weights(0.f, s, pf);
    };
    f32x16 w = scores();
    weigh(w);
    const bool over = !(ls <= E::kMaxWeight);
    if (__any(over)) {
      const bool up = ((int)over | __shfl_xor((int)over, 32, 64)) != 0;  // (every lane takes part in the exchange)
      w = scores();  // (again: kept, they would cost every step sixteen registers)
      float mx = w[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, w[i]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = up ? fmaxf(m_i, mx * p.sl2e) : m_i;
      const float a = mn == m_i ? 1.f : fast_exp2(m_i - mn);
      l_i *= a;
      l_exact *= a;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= a;
      m_i = mn;
      weigh(w);
    }
    if (SAVE) {
#pragma unroll
      for (int i = 0; i < 16; ++i) l_exact += w[i];
    }
    l_i += ls;
    auto vread = [&](int kst, int db) -> u32x4 {
      const bits16* vr = vt + 16 * kst * N;
      return __builtin_shufflevector(lds_read_tr4(vr + voff[0][db]), lds_read_tr4(vr + voff[1][db]), 0, 1, 2, 3);
    };
    if (MASK) {
      uint32_t top = 0;
#pragma unroll
      for (int kst = 0; kst < 2; ++kst)
#pragma unroll
        for (int db = 0; db < DB; ++db) top = max_magnitude(top, vread(kst, db));
      if (__any(not_finite<E>(top) != 0)) {
        hidden = true;
#pragma unroll
        for (int kst = 0; kst < 2; ++kst)
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db] = E::mma(finite_only<E>(vread(kst, db)), pf[kst], o[db]);
        return;
      }
    }
#pragma unroll
    for (int kst = 0; kst < 2; ++kst)
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = E::mma(vread(kst, db), pf[kst], o[db]);
  };

  const int nkv = (kv_end + BKV - 1) / BKV;
  const int nfull = min(nkv, min(q0w + 1, T) / BKV);  // tiles below this wave's first query
  issue_tile(0, 0);
  wait_vmcnt0();
  __syncthreads();
  int j = 0;
  for (; j < nfull; ++j) {
    if (j + 1 < nkv) issue_tile((j + 1) * BKV, (j + 1) & 1);
    const bits16* kt = smem + (j & 1) * 2 * TILE;
#pragma unroll
    for (int st = 0; st < BKV / 32; ++st)
      step(kt + st * 32 * N, kt + TILE + st * 32 * N, j * BKV + 32 * st, std::false_type{});
    wait_vmcnt0();
    __syncthreads();
  }
  for (; j < nkv; ++j) {
    if (j + 1 < nkv) issue_tile((j + 1) * BKV, (j + 1) & 1);
    const bits16* kt = smem + (j & 1) * 2 * TILE;
#pragma unroll
    for (int st = 0; st < BKV / 32; ++st) {
      const int kb0 = j * BKV + st * 32;
      if (kb0 <= q0w + 31) step(kt + st * 32 * N, kt + TILE + st * 32 * N, kb0, std::true_type{});
    }
    wait_vmcnt0();
    __syncthreads();
  }

  if (hidden) {  // wave-uniform
    for (int key = nfull * BKV; key < min(T, q0w + 32); ++key)
#pragma unroll
      for (int db = 0; db < DB; ++db)
        add_not_finite<E>(o[db], vg + (size_t)key * p.v_tok + 32 * db + 4 * h, key <= q0w + c);
  }

  // Normalise, write lse and stage O^T (lane = query) as rows for 16-byte stores.
  bits16* stg = smem + wave * 32 * OP;
  const float inv = 1.0f / (l_i + __shfl_xor(l_i, 32, 64));
  if (SAVE) {
    const float l = l_exact + __shfl_xor(l_exact, 32, 64);
    if (h == 0 && q0w + c < T) p.lse[(size_t)head * p.total + sg.start + q0w + c] = (m_i + __log2f(l)) * kLn2;
  }
  auto store = [&](bits16* out, auto rest_tag) {
    constexpr bool REST = decltype(rest_tag)::value;  // what the rounding leaves
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = o[db][4 * r4 + e] * inv;
        u32x2 w = {E::pack(x[0], x[1]), E::pack(x[2], x[3])};
        if (REST)
          w = u32x2{E::pack(x[0] - E::lo(w[0]), x[1] - E::hi(w[0])), E::pack(x[2] - E::lo(w[1]), x[3] - E::hi(w[1]))};
        *reinterpret_cast<u32x2*>(stg + c * OP + 32 * db + 8 * r4 + 4 * h) = w;
      }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 32 * CH / 64; ++it) {
      const int id = lane + 64 * it, row = id / CH, dc = id % CH;
      if (q0w + row < T)
        st16(out + ((size_t)(sg.start + q0w + row) * p.Hq + head) * N + dc * 8,
             *reinterpret_cast<const u32x4*>(stg + row * OP + dc * 8));
    }
  };
  store(p.o, std::false_type{});
  if (SAVE) {
    __syncthreads();
    store(p.o_rest, std::true_type{});
  }
}

// ---------------------------------------------------------------------------
// dQ: the forward's work list and key tiles. S^T = K Q^T and dP^T = V dO^T, the
// accumulators of the latter starting from -delta (four copies of each query's
// in LDS, read into the registers), dQ^T += K^T dS^T. delta is formed here, from the
// dO rows that are held anyway, and left for the dK/dV kernel (a launch of its own
// for it took 13 us at 26000 tokens, 8 heads of 64, 26 at 16384, 16 of 128).
//
// A sequence's first query sees one key, whose weight is 1 whatever the score:
// its ds is 0, set so rather than left to the difference of two roundings.
// ---------------------------------------------------------------------------
template <class E, int N>
__global__ __launch_bounds__(256, N <= 64 ? 3 : N == 256 ? 1 : 2) void grouped_dq_kernel(GroupedParams p) {
  constexpr int BKV = 64;
  constexpr int CH = N / 8, KS = N / 16, DB = N / 32;
  constexpr int TILE = BKV * N;
  constexpr int OP = N + 8;
  constexpr int SM_LOOP = 4 * TILE * 2, SM_STAT = 4 * 4 * 32 * 16, SM_OUT = 4 * 32 * OP * 2;  // bytes
  constexpr int SMEM = SM_LOOP + SM_STAT > SM_OUT ? SM_LOOP + SM_STAT : SM_OUT;
  __shared__ __attribute__((aligned(16))) unsigned char smem_raw[SMEM];
  bits16* smem = reinterpret_cast<bits16*>(smem_raw);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.Hq / p.Hkv, hw = heads_per_wg(G), BT = 128 / hw, NH = p.Hq / hw;
  const HeadGroup hg = head_group(blockIdx.x % NH, p.Hkv, G, hw);
  const Segment sg = find_segment<true>(p.cu, p.nseq, p.total, BT, blockIdx.x / NH);
  const int T = sg.len, b0 = sg.blk * BT;
  if (b0 >= T) return;
  if (!sg.live) {
    zero_rows<N>(p.dq, sg.start + b0, sg.start + min(b0 + BT, T), hg.q0, hw, p.Hq);
    return;
  }
  const int c = lane & 31, h = lane >> 5;
  const int head = hg.q0 + wave % hw;
  const int q0w = b0 + wave / hw * 32;
  const int kv_end = min(T, b0 + BT);
  const bits16* kg = p.k + (size_t)sg.start * p.k_tok + (size_t)hg.kv * p.k_head;
  const bits16* vg = p.v + (size_t)sg.start * p.v_tok + (size_t)hg.kv * p.v_head;

  u32x4 qf[KS], df[KS];
  const int tq = sg.start + min(q0w + c, T - 1);
  {
    const bits16* qr = p.q + (size_t)tq * p.q_tok + (size_t)head * p.q_head + 8 * h;
    const bits16* dr = p.dO + ((size_t)tq * p.Hq + head) * N + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = ld16(qr + 16 * ks);
      df[ks] = ld16(dr + 16 * ks);
    }
  }
  const float nl = -p.lse_in[(size_t)head * p.total + tq] * kLog2e;
  f32x4* stat = reinterpret_cast<f32x4*>(smem_raw + SM_LOOP) + wave * 128;
  {
    // This lane has half of the row; the other half is lane ^ 32's.
    const bits16* orow = p.o + ((size_t)tq * p.Hq + head) * N + 8 * h;
    const bits16* rest = p.o_rest + ((size_t)tq * p.Hq + head) * N + 8 * h;
    float d = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const u32x4 a = ld16(orow + 16 * ks), b = ld16(rest + 16 * ks);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d = __builtin_fmaf(E::lo(df[ks][e]), E::lo(a[e]) + E::lo(b[e]), d);
        d = __builtin_fmaf(E::hi(df[ks][e]), E::hi(a[e]) + E::hi(b[e]), d);
      }
    }
    d += __shfl_xor(d, 32, 64);
    if (h == 0 && q0w + c < T) p.delta[(size_t)head * p.total + tq] = d;
    const float nd = -d;
#pragma unroll
    for (int j = 0; j < 2; ++j) stat[(2 * h + j) * 32 + c] = f32x4{nd, nd, nd, nd};
  }
  TileLoad<N, BKV> tl;
  tl.init(wave, lane);
  const uint32_t smem_b = lds_addr(smem);
  auto issue_tile = [&](int j0, int stage) {
    const uint32_t at = smem_b + (uint32_t)(stage * 2 * TILE) * 2u;
    tl.issue(kg, p.k_tok, j0, T, at, wave);
    tl.issue(vg, p.v_tok, j0, T, at + TILE * 2u, wave);
  };
  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = zero16();

  const int g16 = lane >> 4, i16 = lane & 15;
  const int tr_row = 4 * h + (i16 >> 2), tr_col = 16 * (g16 & 1) + 4 * (i16 & 3);
  int koff[KS], toff[2][DB];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = swz_off<CH>(c, 16 * ks + 8 * h);
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int db = 0; db < DB; ++db) toff[x][db] = swz_off<CH>(tr_row + 8 * x, 32 * db + tr_col);

  auto step = [&](const bits16* kt, const bits16* vt, int kb0, auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    f32x16 s = zero16(), dp;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 a = stat[j * 32 + c];
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * j + e] = a[e];
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = E::mma(*reinterpret_cast<const u32x4*>(kt + koff[ks]), qf[ks], s);
      dp = E::mma(*reinterpret_cast<const u32x4*>(vt + koff[ks]), df[ks], dp);
    }
    const int qq = q0w + c;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float w = fast_exp2(__builtin_fmaf(s[i], p.sl2e, nl));
      float d = w * dp[i];
      if (MASK) {
        const int key = kb0 + 8 * (i >> 2) + 4 * h + (i & 3);
        if (key > qq || key >= T || qq == 0) d = 0.f;
      }
      s[i] = d;
    }
    u32x4 sf[2];
#pragma unroll
    for (int kst = 0; kst < 2; ++kst)
#pragma unroll
      for (int e = 0; e < 4; ++e) sf[kst][e] = E::pack(s[8 * kst + 2 * e], s[8 * kst + 2 * e + 1]);
    // On the diagonal, where a sequence's first rows have all their keys, what rounding ds
    // left goes in as well: few keys leave few errors to even out (sequences of 1 to 5
    // tokens: dq and dk 2.5e-3 off their norms without it, 1.9e-3 with it, 1.7e-3 if
    // nothing but the outputs were rounded; 1% of forward and backward at 1100 tokens).
    u32x4 rest[2];
    if (MASK) {
#pragma unroll
      for (int kst = 0; kst < 2; ++kst)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = sf[kst][e];
          rest[kst][e] = E::pack(s[8 * kst + 2 * e] - E::lo(w), s[8 * kst + 2 * e + 1] - E::hi(w));
        }
    }
#pragma unroll
    for (int kst = 0; kst < 2; ++kst)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const bits16* kr = kt + 16 * kst * N;
        const u32x4 kf = __builtin_shufflevector(lds_read_tr4(kr + toff[0][db]), lds_read_tr4(kr + toff[1][db]), 0, 1, 2, 3);
        dq[db] = E::mma(kf, sf[kst], dq[db]);
        if (MASK) dq[db] = E::mma(kf, rest[kst], dq[db]);
      }
  };

  const int nkv = (kv_end + BKV - 1) / BKV;
  const int nfull = min(nkv, min(q0w + 1, T) / BKV);
  issue_tile(0, 0);
  wait_vmcnt0();
  __syncthreads();
  int j = 0;
  for (; j < nfull; ++j) {
    if (j + 1 < nkv) issue_tile((j + 1) * BKV, (j + 1) & 1);
    const bits16* kt = smem + (j & 1) * 2 * TILE;
#pragma unroll
    for (int st = 0; st < 2; ++st)
      step(kt + st * 32 * N, kt + TILE + st * 32 * N, j * BKV + 32 * st, std::false_type{});
    wait_vmcnt0();
    __syncthreads();
  }
  for (; j < nkv; ++j) {
    if (j + 1 < nkv) issue_tile((j + 1) * BKV, (j + 1) & 1);
    const bits16* kt = smem + (j & 1) * 2 * TILE;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int kb0 = j * BKV + st * 32;
      if (kb0 <= q0w + 31) step(kt + st * 32 * N, kt + TILE + st * 32 * N, kb0, std::true_type{});
    }
    wait_vmcnt0();
    __syncthreads();
  }

  bits16* stg = smem + wave * 32 * OP;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x16& a = dq[db];
      *reinterpret_cast<u32x2*>(stg + c * OP + 32 * db + 8 * r4 + 4 * h) =
          u32x2{E::pack(a[4 * r4] * p.scale, a[4 * r4 + 1] * p.scale), E::pack(a[4 * r4 + 2] * p.scale, a[4 * r4 + 3] * p.scale)};
    }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 32 * CH / 64; ++it) {
    const int id = lane + 64 * it, row = id / CH, dc = id % CH;
    if (q0w + row < T)
      st16(p.dq + ((size_t)(sg.start + q0w + row) * p.Hq + head) * N + dc * 8,
           *reinterpret_cast<const u32x4*>(stg + row * OP + dc * 8));
  }
}

// ---------------------------------------------------------------------------
// dK, dV: one workgroup per (segment, key head, 128 keys), wave w its keys
// 32 w .. 32 w + 31; the query tiles of every head of the group stream through
// LDS, so the sum over the group stays in the accumulators (fixed order, no
// atomics). The tiles, head after head, are cut into p.parts equal runs for as many
// workgroups where the key blocks alone are too few to fill the card and even out
// the causal blocks' lengths (see dkdv_parts); their fp32 sums are then added, in
// order, by a second launch. S = Q K^T and dP = dO V^T with the key on the lane; the start values
// -lse / scale and -delta come from LDS rows. dV^T += dO^T P, dK^T += Q^T dS.
// ---------------------------------------------------------------------------
template <class E, int N>
__global__ __launch_bounds__(256, N <= 64 ? 3 : N == 128 ? 2 : 1) void grouped_dkdv_kernel(GroupedParams p) {
  constexpr int BK = 128;                 // keys per workgroup
  constexpr int BQ = N >= 128 ? 32 : 64;  // queries per LDS tile
  constexpr int CH = N / 8, KS = N / 16, DB = N / 32;
  constexpr int TILE = BQ * N;
  constexpr int OP = N + 8;
  constexpr int SM_LOOP = 2 * 2 * TILE * 2 + 2 * 2 * BQ * 4;  // bytes
  constexpr int SM_V = 4 * KS * 64 * 16;  // each wave's V^T fragments, [wave][ks][lane]
  constexpr int SM_OUT = 4 * 32 * OP * 2;
  constexpr int SMEM = SM_LOOP + SM_V > SM_OUT ? SM_LOOP + SM_V : SM_OUT;
  __shared__ __attribute__((aligned(16))) unsigned char smem[SMEM];
  bits16* tiles = reinterpret_cast<bits16*>(smem);                         // [stage][Q | dO]
  float* statf = reinterpret_cast<float*>(smem + 2 * 2 * TILE * 2);        // [stage][-lse / scale | -delta][query]
  u32x4* vown = reinterpret_cast<u32x4*>(smem + SM_LOOP);

  const int G = p.Hq / p.Hkv, kv = blockIdx.x % p.Hkv, vp = blockIdx.x / p.Hkv;
  const int part = vp % p.parts;
  const Segment sg = find_segment<false>(p.cu, p.nseq, p.total, BK, vp / p.parts);
  const int T = sg.len, k0 = sg.blk * BK;
  if (k0 >= T) return;
  if (!sg.live) {
    if (part != 0) return;
    zero_rows<N>(p.dk, sg.start + k0, sg.start + min(k0 + BK, T), kv, 1, p.Hkv);
    zero_rows<N>(p.dv, sg.start + k0, sg.start + min(k0 + BK, T), kv, 1, p.Hkv);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int kw0 = k0 + wave * 32;

  u32x4 kf[KS];
  u32x4* vw = vown + wave * KS * 64;
  {
    const size_t t = sg.start + min(kw0 + c, T - 1);
    const bits16* kr = p.k + t * p.k_tok + (size_t)kv * p.k_head + 8 * h;
    const bits16* vr = p.v + t * p.v_tok + (size_t)kv * p.v_head + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[ks] = ld16(kr + 16 * ks);
      vw[ks * 64 + lane] = ld16(vr + 16 * ks);
    }
  }

  TileLoad<N, BQ> tl;
  tl.init(wave, lane);
  const uint32_t tiles_b = lds_addr(tiles);
  const float inv_sl = -1.0f / p.scale;
  float st_l = 0.f, st_d = 0.f;
  auto issue_tile = [&](int head, int q0, int stage) {
    const uint32_t at = tiles_b + (uint32_t)(stage * 2 * TILE) * 2u;
    tl.issue(p.q + (size_t)sg.start * p.q_tok + (size_t)head * p.q_head, p.q_tok, q0, T, at, wave);
    tl.issue(p.dO + ((size_t)sg.start * p.Hq + head) * N, (int64_t)p.Hq * N, q0, T, at + TILE * 2u, wave);
    if (tid < BQ) {
      const size_t t = (size_t)head * p.total + sg.start + min(q0 + tid, T - 1);
      st_l = p.lse_in[t];
      st_d = p.delta[t];
    }
  };
  // After wait_vmcnt0(): the statistics have landed with their tile.
  auto publish = [&](int stage) {
    if (tid < BQ) {
      statf[stage * 2 * BQ + tid] = st_l * inv_sl;
      statf[stage * 2 * BQ + BQ + tid] = -st_d;
    }
  };

  f32x16 dv[DB], dk[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dv[db] = dk[db] = zero16();

  const int g16 = lane >> 4, i16 = lane & 15;
  const int tr_row = 4 * h + (i16 >> 2), tr_col = 16 * (g16 & 1) + 4 * (i16 & 3);
  // (Recomputed per use: registers bound the workgroups per CU.)
  auto kofs = [&](int ks) { return swz_off<CH>(c, 16 * ks + 8 * h); };
  auto tofs = [&](int x, int db) { return swz_off<CH>(tr_row + 8 * x, 32 * db + tr_col); };

  // One 32-query step of the tile at q0.
  auto step = [&](const bits16* qt, const bits16* dt, const float* stf, int qs0, auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    f32x16 s, dp;
    const float* sl = stf + 4 * h;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(sl + 8 * j);
      const f32x4 b = *reinterpret_cast<const f32x4*>(sl + BQ + 8 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[4 * j + e] = a[e];
        dp[4 * j + e] = b[e];
      }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = E::mma(*reinterpret_cast<const u32x4*>(qt + kofs(ks)), kf[ks], s);
      dp = E::mma(*reinterpret_cast<const u32x4*>(dt + kofs(ks)), vw[ks * 64 + lane], dp);
    }
    const int key = kw0 + c;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float w = fast_exp2(s[i] * p.sl2e);
      float d = w * dp[i];
      if (MASK) {
        const int q = qs0 + 8 * (i >> 2) + 4 * h + (i & 3);
        if (key > q || q >= T) w = d = 0.f;
        if (q == 0) d = 0.f;  // one key: see dQ
      }
      s[i] = w;
      dp[i] = d;
    }
    u32x4 pb[2], sb[2];
#pragma unroll
    for (int kst = 0; kst < 2; ++kst)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pb[kst][e] = E::pack(s[8 * kst + 2 * e], s[8 * kst + 2 * e + 1]);
        sb[kst][e] = E::pack(dp[8 * kst + 2 * e], dp[8 * kst + 2 * e + 1]);
      }
    u32x4 rest[2];  // what rounding ds left: see dQ
    if (MASK) {
#pragma unroll
      for (int kst = 0; kst < 2; ++kst)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = sb[kst][e];
          rest[kst][e] = E::pack(dp[8 * kst + 2 * e] - E::lo(w), dp[8 * kst + 2 * e + 1] - E::hi(w));
        }
    }
#pragma unroll
    for (int kst = 0; kst < 2; ++kst)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const int rb = 16 * kst * N, o0 = rb + tofs(0, db), o1 = rb + tofs(1, db);
        const u32x4 dT = __builtin_shufflevector(lds_read_tr4(dt + o0), lds_read_tr4(dt + o1), 0, 1, 2, 3);
        const u32x4 qT = __builtin_shufflevector(lds_read_tr4(qt + o0), lds_read_tr4(qt + o1), 0, 1, 2, 3);
        dv[db] = E::mma(dT, pb[kst], dv[db]);
        dk[db] = E::mma(qT, sb[kst], dk[db]);
        if (MASK) dk[db] = E::mma(qT, rest[kst], dk[db]);
      }
  };

  // Tiles of a head from the last queries down to the block's own keys (every
  // workgroup of a head reads the same tile at about the same time), head by
  // head. Tiles 0 .. nfull-1 lie above the block's keys; the first may run past
  // the sequence's end.
  const int nq = (T - k0 + BQ - 1) / BQ, nfull = nq - BK / BQ;
  const bool ragged = (T - k0) % BQ != 0;
  auto row_of = [&](int it) { return k0 + (nq - 1 - it) * BQ; };
  // This part's run: tiles first .. last - 1 of the nq * G.
  const int n = nq * G, first = (int)((int64_t)n * part / p.parts), last = (int)((int64_t)n * (part + 1) / p.parts);
  int g = first / nq, left = last - first, stage = 0;
  auto tile = [&](int it, auto masked_tag) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const int q0 = row_of(it);
    const bool wrap = it + 1 == nq, more = --left > 0;
    if (more) issue_tile(kv * G + g + (wrap ? 1 : 0), row_of(wrap ? 0 : it + 1), stage ^ 1);
    const bits16* qt = tiles + stage * 2 * TILE;
    const bits16* dt = qt + TILE;
    const float* stf = statf + stage * 2 * BQ;
#pragma unroll
    for (int sub = 0; sub < BQ / 32; ++sub) {
      const int qs0 = q0 + 32 * sub;
      if (MASKED && (qs0 + 31 < kw0 || qs0 >= T)) continue;  // wave-uniform: nothing to add
      step(qt + 32 * sub * N, dt + 32 * sub * N, stf + 32 * sub, qs0, masked_tag);
      // Keeps the next step's S and dP from being scheduled into this one.
      if (!MASKED) __builtin_amdgcn_sched_barrier(0);
    }
    wait_vmcnt0();
    if (more) publish(stage ^ 1);
    __syncthreads();
    stage ^= 1;
  };
  if (left > 0) {
    issue_tile(kv * G + g, row_of(first - g * nq), 0);
    wait_vmcnt0();
    publish(0);
    __syncthreads();
  }
  int it = first - g * nq;
  while (left > 0) {
    const int end = min(nq, it + left), full = min(nfull, end);
    if (it == 0 && nfull > 0 && ragged) tile(it++, std::true_type{});
    for (; it < full; ++it) tile(it, std::false_type{});
    for (; it < end; ++it) tile(it, std::true_type{});
    ++g;
    it = 0;
  }

  if (p.parts > 1) {
    // fp32 sums: (part, dk | dv, token, key head, N); a lane has 4 columns at a time.
    float* out = p.sums + (((size_t)part * 2 * p.total + sg.start + kw0 + c) * p.Hkv + kv) * N + 4 * h;
    if (kw0 + c < T) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          float* at = out + 32 * db + 8 * r4;
          *reinterpret_cast<f32x4*>(at) = f32x4{dk[db][4 * r4], dk[db][4 * r4 + 1], dk[db][4 * r4 + 2], dk[db][4 * r4 + 3]};
          *reinterpret_cast<f32x4*>(at + (size_t)p.total * p.Hkv * N) =
              f32x4{dv[db][4 * r4], dv[db][4 * r4 + 1], dv[db][4 * r4 + 2], dv[db][4 * r4 + 3]};
        }
    }
    return;
  }
  bits16* stg = reinterpret_cast<bits16*>(smem) + wave * 32 * OP;
  auto store = [&](const f32x16 (&a)[DB], float f, bits16* out) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *reinterpret_cast<u32x2*>(stg + c * OP + 32 * db + 8 * r4 + 4 * h) =
            u32x2{E::pack(a[db][4 * r4] * f, a[db][4 * r4 + 1] * f), E::pack(a[db][4 * r4 + 2] * f, a[db][4 * r4 + 3] * f)};
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 32 * CH / 64; ++u) {
      const int id = lane + 64 * u, row = id / CH, dc = id % CH;
      if (kw0 + row < T)
        st16(out + ((size_t)(sg.start + kw0 + row) * p.Hkv + kv) * N + dc * 8,
             *reinterpret_cast<const u32x4*>(stg + row * OP + dc * 8));
    }
    __syncthreads();
  };
  store(dv, 1.0f, p.dv);
  store(dk, p.scale, p.dk);
}

// The sums of the parts, eight elements a thread, to dk (times scale) and dv. Rows
// of no sequence have no sums: they stay as the first launch zeroed them.
template <class E>
__global__ __launch_bounds__(256) void grouped_dkdv_join_kernel(GroupedParams p, int N) {
  const size_t each = (size_t)p.total * p.Hkv * N, at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= each) return;
  const int t = (int)(at / ((size_t)p.Hkv * N));
  if (t < p.cu[0] || t >= p.cu[p.nseq]) return;
  f32x4 a[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = zero4();
  for (int part = 0; part < p.parts; ++part) {
    const float* s = p.sums + (size_t)part * 2 * each + at;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] += *reinterpret_cast<const f32x4*>(s + (i >> 1) * each + (i & 1) * 4);
  }
  a[0] *= p.scale;
  a[1] *= p.scale;
  st16(p.dk + at, u32x4{E::pack(a[0][0], a[0][1]), E::pack(a[0][2], a[0][3]), E::pack(a[1][0], a[1][1]), E::pack(a[1][2], a[1][3])});
  st16(p.dv + at, u32x4{E::pack(a[2][0], a[2][1]), E::pack(a[2][2], a[2][3]), E::pack(a[3][0], a[3][1]), E::pack(a[3][2], a[3][3])});
}

// Calls k(std::integral_constant<int, N>) for a supported head width.
template <class F>
hipError_t by_width(int N, F k) {
  if (N == 32)
    k(std::integral_constant<int, 32>{});
  else if (N == 64)
    k(std::integral_constant<int, 64>{});
  else if (N == 128)
    k(std::integral_constant<int, 128>{});
  else if (N == 256)
    k(std::integral_constant<int, 256>{});
  else
    return hipErrorInvalidValue;
  return hipGetLastError();
}

unsigned query_grid(const GroupedParams& p) {
  const int G = p.Hq / p.Hkv, hw = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
  return (unsigned)virtual_blocks(p.total, p.nseq, 128 / hw) * (unsigned)(p.Hq / hw);
}

}  // namespace

// Parts of a key block's query tiles, at most eight: as many as fill the card, with
// four tiles each at least; or as many as give its slots three workgroups each, which
// evens out the causal blocks' lengths, where a part has 64 tiles at least, whose
// time makes up for the sums' way through memory. (T = 8192 x 2, 16 / 4 heads of 128,
// dK/dV with the join: 1 part 1394 us, 2, 3, 4 parts 948, 921, 910; 24 sequences of
// 1100 on average, 8 / 4 heads of 64, 17 tiles a block: 1 part 147 us, 4 parts 199.)
int dkdv_parts(int total, int nseq, int Hq, int Hkv, int N) {
  const int64_t slots = 256 * (N <= 64 ? 3 : N == 128 ? 2 : 1), blocks = (int64_t)(total / 128 + nseq) * Hkv;
  const int64_t tiles = (int64_t)(total / nseq) * (Hq / Hkv) / (2 * (N >= 128 ? 32 : 64));  // of a block, on average
  const int64_t fill = slots / blocks < tiles / 4 ? slots / blocks : tiles / 4;
  const int64_t even = (3 * slots + blocks - 1) / blocks, parts = even < tiles / 64 ? even : tiles / 64;
  const int64_t n = fill > parts ? fill : parts;
  return n < 1 ? 1 : n > 8 ? 8 : (int)n;
}

hipError_t launch_grouped_join(const GroupedParams& p, int N, hipStream_t s) {
  const size_t threads = (size_t)p.total * p.Hkv * N / 8;
  hipLaunchKernelGGL(grouped_dkdv_join_kernel<Bf16>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, p, N);
  return hipGetLastError();
}

hipError_t launch_grouped_fwd(const GroupedParams& p, int N, bool fp16, hipStream_t s) {
  const dim3 grid(query_grid(p));
  return by_width(N, [&](auto n) {
    if (fp16)
      hipLaunchKernelGGL((grouped_fwd_kernel<Fp16, n.value, false>), grid, dim3(256), 0, s, p);
    else if (p.lse == nullptr)
      hipLaunchKernelGGL((grouped_fwd_kernel<Bf16, n.value, false>), grid, dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((grouped_fwd_kernel<Bf16, n.value, true>), grid, dim3(256), 0, s, p);
  });
}

hipError_t launch_grouped_dq(const GroupedParams& p, int N, hipStream_t s) {
  const dim3 grid(query_grid(p));
  return by_width(N, [&](auto n) { hipLaunchKernelGGL((grouped_dq_kernel<Bf16, n.value>), grid, dim3(256), 0, s, p); });
}

hipError_t launch_grouped_dkdv(const GroupedParams& p, int N, hipStream_t s) {
  const dim3 grid((unsigned)virtual_blocks(p.total, p.nseq, 128) * (unsigned)(p.Hkv * p.parts));
  return by_width(N, [&](auto n) { hipLaunchKernelGGL((grouped_dkdv_kernel<Bf16, n.value>), grid, dim3(256), 0, s, p); });
}

}  // namespace mea
