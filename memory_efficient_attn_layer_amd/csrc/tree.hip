// Attention of n new tokens per sequence over a paged cache on gfx950 MFMA: one
// token of a decoding step (n = 1), or a drafted tree whose tokens see their
// ancestors. The new tokens' k and v are already the last n rows of the cache:
//   o_i = sum_r w_ir v_r / sum_r w_ir,  w_ir = exp(scale q_i . k_r)  over the rows
//   r < len - n, and r = len - n + j where mask[i][j];  0 where there is none.
//
// Bound by reading the cache once from HBM: the rows of a key head are read for
// all its R = n * G query rows together (row i * G + g, G query heads to a key
// head), 32 of them to a wave, on v_mfma_f32_32x32x16 with the query on the lane (the
// forms of attn_fwd.hip, S^T = K Q^T, O^T += V^T P^T). Few query rows leave the keys
// to be split (flash decoding): into chunks, one workgroup each, and over KG key
// groups of the workgroup, which walk alternate tiles; RW waves of a group take
// 32 query rows each of the tiles they share. Tiles stream into a ring in LDS that
// is the group's own. A wave alone in its group (RW = 1) waits for its own loads
// only, no barrier in the loop, and the other waves' loads stay in flight meanwhile;
// sharing waves pass one barrier per tile. Two workgroups a CU, two waves a SIMD where
// their registers allow it, or one of twice the waves: a wave alone runs its products and exponentials one
// after the other.
//
// Chunks: the host knows capacities, not lengths. Every workgroup reads all
// lengths and settles the chunk size by itself: where sequences are few, the smallest,
// in whole turns of the waves, that gives at most as many chunks as run at one time,
// so that they end together. Several chunks of a sequence leave fp32 sums, which the second launch
// adds in order.
//
// Pages: the chunk's table entries are read once into LDS; pages hold sixteen rows
// or a multiple, so that every load instruction lies in one page. Rows of pages
// outside the pool are masked.
#include <type_traits>

#include "elem.cuh"
#include "grouped.h"

namespace mea {

namespace {

constexpr int kMaxChunk = 8192;             // keys
constexpr int kTab = kMaxChunk / 16 + 2;    // its table entries at 16 rows a page
constexpr int kSeenPitch = kMaxTree / 32 + 1;  // words of a mask's row (the last is not used)

// RW waves share a tile, KG groups of them run; rings of NS tiles, 64 KB and two
// workgroups a CU. Four waves a tile: tiles and rings of twice the size and one
// workgroup a CU, whose two groups join their sums in LDS, so that half as many go
// through memory. (N = 128, 16 sequences of up to 4096 rows, 32 tokens: 41.0 us with two
// workgroups of one group, 38.6 so, 37.4 with four tiles of half the size; one of
// 131072 rows, 64 tokens: 133.2, 132.0, 135.4.)
template <int N, int RW>
struct Tile {
  static constexpr int ST = (N >= 128 ? 1 : 128 / N) * (RW == 4 && N < 256 ? 2 : 1);  // 32-key steps
  static constexpr int KEYS = 32 * ST, ELEMS = KEYS * N;
  static constexpr int KG = N == 256 ? 1 : 2, NS = 2;
  static constexpr int WAVES = RW * KG, LOADS = ELEMS / 8 / 64 / RW;
  static constexpr int RING = NS * 2 * ELEMS;  // [stage][K | V]
  static constexpr int TURN = KEYS * KG;  // keys of one turn of the workgroup
  static constexpr int SLOTS = RW == 4 ? 256 : 512;  // workgroups at one time
};

// s_waitcnt vmcnt(n), and nothing that reads or writes memory moves across it.
template <int n>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// (By a permute, not a scalar register: the loop's counts in scalars cost the kernel spills.)
__device__ __forceinline__ int wave_add(int v) { return __shfl(wave_scan(v), 63, 64); }

constexpr int kLeast = 2048;      // keys of a chunk where sequences are many
// Beyond so many, or where their rows could be 2^35 (the count of them in 32 bits),
// every sequence has the same number of items, of kMaxChunk keys.
constexpr int kManySeqs = 4096;

// The chunk size, and the sequence and chunk that are item `item` of a head.
struct Chunk {
  int size, seq, chunk, count;  // seq < 0: no such item; count: the sequence's chunks (0 where it has no row)
};
// want, least, full: of TreeGrid; turn: granule of the size.
__device__ __forceinline__ Chunk find_chunk(const PagedCache& c, int want, int turn, int least, int full, int item) {
  const int lane = threadIdx.x & 63;
  auto len = [&](int s) { return min(max(c.lengths[s], 0), c.max_pages << c.lg_page); };
  Chunk r;
  if (want == 0) {
    r.size = kMaxChunk;
    r.seq = item / full;
    r.chunk = item - r.seq * full;
    r.count = r.seq < c.seqs ? (len(r.seq) + kMaxChunk - 1) / kMaxChunk : 0;
    if (r.seq >= c.seqs || r.chunk >= max(r.count, 1)) r.seq = -1;
    return r;
  }
  // Lane l holds sequences l * per .. l * per + per - 1; the first in a register.
  const int per = (c.seqs + 63) >> 6, mine0 = lane * per, len0 = mine0 < c.seqs ? len(mine0) : 0;
  auto sum = [&](auto f) {
    int v = mine0 < c.seqs ? f(len0) : 0;
    for (int s = mine0 + 1; s < min(mine0 + per, c.seqs); ++s) v += f(len(s));
    return v;
  };
  auto whole = [&](int keys) { return (keys + turn - 1) / turn * turn; };
  auto chunks = [&](int n) { return max((n + r.size - 1) / r.size, 1); };
  // Few sequences: as many chunks as run at one time. Many: four times as many, which
  // even out the rounds. (Sums of keys in units of 16, so that they fit 32 bits.)
  const bool few = 2 * c.seqs <= want;
  const int total = wave_add(sum([](int n) { return (n + 15) >> 4; })), parts = few ? want : 4 * want;
  r.size = min(max(whole(((total + parts - 1) / parts) << 4), least), kMaxChunk);
  while (few && r.size < kMaxChunk && wave_add(sum(chunks)) > want) r.size = min(whole(r.size + r.size / 16), kMaxChunk);
  // Item -> (sequence, chunk): every sequence has one item at least.
  const int own = sum(chunks), up = wave_scan(own);
  const unsigned long long at = __ballot(up > item);
  r.seq = -1;
  if (at == 0) return r;
  const int l = __ffsll(at) - 1;
  int rest = item - __shfl(up - own, l, 64), s = l;
  if (per > 1) {
    s = l * per + lane;
    const int n = lane < per && s < c.seqs ? chunks(len(s)) : 0, to = wave_scan(n);
    const int k = __ffsll(__ballot(to > rest)) - 1;
    rest -= __shfl(to - n, k, 64);
    s = l * per + k;
  }
  r.seq = __builtin_amdgcn_readfirstlane(s);
  r.chunk = __builtin_amdgcn_readfirstlane(rest);
  r.count = __builtin_amdgcn_readfirstlane((len(r.seq) + r.size - 1) / r.size);
  return r;
}

template <class E, int N, int RW>
__global__ __launch_bounds__((64 * Tile<N, RW>::WAVES), RW == 1 || N == 256 ? 1 : 2) void tree_attn_kernel(TreeParams p) {
  using T = Tile<N, RW>;
  constexpr int ST = T::ST, WAVES = T::WAVES, LOADS = T::LOADS, KG = T::KG, NS = T::NS;
  constexpr int CH = N / 8, KS = N / 16, DB = N / 32;
  static_assert(KG == 1 || KG * T::RING >= RW * DB * 16 * 64 * 2, "the exchange of one group's fp32 sums fits the rings");
  __shared__ __attribute__((aligned(16))) bits16 smem_all[KG * T::RING];
  __shared__ int tab[kTab];
  __shared__ uint32_t seen_s[RW * 32 * kSeenPitch];
  __shared__ float xm[KG > 1 ? RW * 64 : 1], xl[KG > 1 ? RW * 64 : 1];

  const PagedCache& cc = p.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave % RW, kg = wave / RW;
  const int c = lane & 31, h = lane >> 5;
  const int G = p.Hq / cc.Hkv, R = p.n * G;
  // Key heads fastest, then the row groups that read the same rows, then chunks.
  const int kv = blockIdx.x % cc.Hkv, grp = blockIdx.x / cc.Hkv, item = grp / p.row_groups;
  const Chunk ck = find_chunk(cc, p.want, T::TURN, p.least, p.full, item);
  if (ck.seq < 0) return;
  const int s = ck.seq;
  const int len = __builtin_amdgcn_readfirstlane(min(max(cc.lengths[s], 0), cc.max_pages << cc.lg_page));
  const int ctx = max(len - p.n, 0), lead = p.n - (len - ctx);  // lead: tokens in front of a short sequence's rows
  const int k_begin = ck.chunk * ck.size, k_end = min(k_begin + ck.size, len);
  const int r0 = ((grp - item * p.row_groups) * RW + rw) * 32;  // first query row of the wave
  const int tok0 = (grp - item * p.row_groups) * RW * 32 / G;   // first token of the workgroup

  // Query row r = i * G + g: token i, head kv * G + g.
  const int r = min(r0 + c, R - 1), qi = r / G;
  const size_t hq = (size_t)kv * G + (r - qi * G);

  float m_i = -INFINITY, l_i = 0.f;  // l_i: this lane's half of the keys
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();

  if (k_begin < k_end) {  // uniform over the workgroup
    // Table entries of the chunk; whether all of them lie in the pool.
    const int first = k_begin >> cc.lg_page, pages = ((k_end - 1) >> cc.lg_page) - first + 1;
    bool ok = true;
    for (int i = tid; i < pages; i += 64 * WAVES) {
      const int page = cc.table[(size_t)s * cc.max_pages + first + i];
      const bool in = (unsigned)page < (unsigned)cc.pages;
      tab[i] = in ? page : -1;
      ok = ok && in;
    }
    const bool all_in = __syncthreads_and(ok);

    u32x4 qf[KS];
    {
      const bits16* qr = p.q + s * p.q_seq + qi * p.q_tok + (int64_t)hq * p.q_head + 8 * h;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = ld16(qr + 16 * ks);
    }
    const size_t head_page = (size_t)cc.N << cc.lg_page;  // elements of one head's rows of a page
    bits16* ring = smem_all + kg * T::RING;
    const uint32_t ring_b = lds_addr(ring);
    const int nt = (k_end - k_begin + T::KEYS - 1) / T::KEYS;
    // Tile t (of the chunk) into a stage; a load instruction's rows lie in one page,
    // so that it has a uniform base and a lane-constant offset. One of rows past the
    // chunk, or of no page, reads the pool's first rows (the loads in flight are then
    // always the same number).
    uint32_t ld_off[LOADS];  // within the load's sixteen rows (bytes)
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int slot = (rw * LOADS + u) * 64 + lane, row = slot / CH;
      ld_off[u] = (uint32_t)((row & 15) * N + ((slot % CH) ^ chunk_swz<CH>(row)) * 8) * 2u;
    }
    auto issue = [&](int t, int stage) {
      const uint32_t at = ring_b + (uint32_t)(stage * 2 * T::ELEMS) * 2u;
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int w = rw * LOADS + u, key = k_begin + t * T::KEYS + (w * 64 / CH & ~15);  // uniform: first of sixteen rows
        const int page = __builtin_amdgcn_readfirstlane(key < k_end ? tab[(key >> cc.lg_page) - first] : -1);
        const size_t off = page < 0 ? 0 : ((size_t)page * cc.Hkv + kv) * head_page + (size_t)(key & (cc.page - 1)) * N;
        g2lds16_s(cc.k + off, ld_off[u], at + (uint32_t)w * 1024u);
        g2lds16_s(cc.v + off, ld_off[u], at + (uint32_t)T::ELEMS * 2u + (uint32_t)w * 1024u);
      }
    };
    // V rows of a tile that are no rows of the sequence become 0 in LDS: what lies
    // there in the pool may be anything, and their weights are 0.
    auto clear_tail = [&](bits16* vt, int t) {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int slot = (rw * LOADS + u) * 64 + lane, key = k_begin + t * T::KEYS + slot / CH;
        if (key >= k_end || tab[(key >> cc.lg_page) - first] < 0) *reinterpret_cast<u32x4*>(vt + slot * 8) = u32x4{0u, 0u, 0u, 0u};
      }
      wait_lds();
    };

    const int g16 = lane >> 4, i16 = lane & 15;
    const int tr_row = 4 * h + (i16 >> 2), tr_col = 16 * (g16 & 1) + 4 * (i16 & 3);
    int koff[KS], voff[2][DB];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) koff[ks] = swz_off<CH>(c, 16 * ks + 8 * h);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int db = 0; db < DB; ++db) voff[x][db] = swz_off<CH>(tr_row + 8 * x, 32 * db + tr_col);

    // Whether the token qi sees the sixteen rows that this lane has of a step (bit i:
    // key kb0 + 8 (i >> 2) + 4 h + (i & 3)), from the 32 of the step, bit by bit.
    auto visible = [&](int kb0) -> uint32_t {
      const int at = kb0 - ctx + lead;  // token of the first row; below 0: rows that all see
      uint32_t w;
      if (p.mask == nullptr) {
        const int d = qi - at + 1;  // rows that qi sees
        w = d >= 32 ? ~0u : (1u << max(d, 0)) - 1u;
      } else {
        const uint32_t* row = seen_s + (qi - tok0) * kSeenPitch;
        if (at >= 0)
          w = (uint32_t)(((uint64_t)row[(at >> 5) + 1] << 32 | row[at >> 5]) >> (at & 31));
        else
          w = at <= -32 ? ~0u : (row[0] << -at | ((1u << -at) - 1u));
      }
      const int rows = k_end - kb0;
      if (rows < 32) w &= (1u << rows) - 1u;
      w = w >> (4 * h) & 0x0F0F0F0Fu;
      w = (w | w >> 4) & 0x00FF00FFu;
      w = (w | w >> 8) & 0xFFFFu;
      if (!all_in) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = min(kb0 + 8 * (i >> 2) + 4 * h + (i & 3), k_end - 1);
          w &= ~((uint32_t)(tab[(key >> cc.lg_page) - first] < 0) << i);
        }
      }
      return w;
    };

    // One 32-key step, as in the forward of the packed prompts; MASK: some row may
    // be hidden from some query. A query that has seen no key yet has m = -inf.
    bool hidden = false;  // a masked step's V held infinities or NaN, left out there
    auto step = [&](const bits16* kt, const bits16* vt, int kb0, auto mask_tag) {
      constexpr bool MASK = decltype(mask_tag)::value;
      const uint32_t seen = MASK ? visible(kb0) : 0;
      auto scores = [&] {
        f32x16 w = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) w = E::mma(*reinterpret_cast<const u32x4*>(kt + koff[ks]), qf[ks], w);
        if (MASK) {
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = (seen >> i & 1) != 0 ? w[i] : -INFINITY;
        }
        return w;
      };
      f32x16 w = scores();
      u32x4 pf[2];
      float ls;  // sum of the step's weights
      auto weigh = [&](float m) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = fast_exp2(__builtin_fmaf(w[i], p.sl2e, -m));
#pragma unroll
        for (int kst = 0; kst < 2; ++kst)
#pragma unroll
          for (int e = 0; e < 4; ++e) pf[kst][e] = E::pack(w[8 * kst + 2 * e], w[8 * kst + 2 * e + 1]);
        ls = E::add_weights(0.f, w, pf);
      };
      weigh(m_i);
      const bool over = !(ls <= E::kMaxWeight);
      if (__any(over)) {
        const bool up = ((int)over | __shfl_xor((int)over, 32, 64)) != 0;  // (every lane takes part in the exchange)
        w = scores();
        float mx = w[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, w[i]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = up ? fmaxf(m_i, mx * p.sl2e) : m_i;
        const float a = mn == m_i ? 1.f : fast_exp2(m_i - mn);
        l_i *= a;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= a;
        m_i = mn;
        // No key seen: weights exp2(-inf - 0) = 0. (NaN scores stay NaN.)
        weigh(mn == -INFINITY ? 0.f : mn);
      }
      l_i += ls;
      auto vread = [&](int kst, int db) -> u32x4 {
        const bits16* vr = vt + 16 * kst * N;
        return __builtin_shufflevector(lds_read_tr4(vr + voff[0][db]), lds_read_tr4(vr + voff[1][db]), 0, 1, 2, 3);
      };
      bool bad = false;
      if (MASK) {
        uint32_t top = 0;
#pragma unroll
        for (int kst = 0; kst < 2; ++kst)
#pragma unroll
          for (int db = 0; db < DB; ++db) top = max_magnitude(top, vread(kst, db));
        bad = __any(not_finite<E>(top) != 0);
        hidden = hidden || bad;
      }
#pragma unroll
      for (int kst = 0; kst < 2; ++kst)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          u32x4 vf = vread(kst, db);
          if (MASK && bad) vf = finite_only<E>(vf);
          o[db] = E::mma(vf, pf[kst], o[db]);
        }
    };

    // Rows that every query sees: whole steps below free_end.
    const int free_end = all_in ? min(ctx, k_end) : 0;
    const bool idle = r0 >= R;  // no query rows left for this wave
#pragma unroll
    for (int i = 0; i < NS - (RW > 1 ? 1 : 0); ++i) issue(kg + i * KG, i);
    // The mask's rows of the workgroup's tokens, where the chunk has rows of the tree,
    // as bits, while the first tiles are under way.
    if (p.mask != nullptr && k_end > ctx) {
      const unsigned char* mask = p.mask + s * p.mask_seq;
      const int rows = min(((grp - item * p.row_groups) * RW * 32 + RW * 32 - 1) / G, p.n - 1) - tok0 + 1;
      for (int j = lane; j - lane < p.n; j += 64)
        for (int i = wave; i < rows; i += 4 * WAVES) {
          unsigned char b[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) b[u] = mask[(int64_t)(tok0 + min(i + u * WAVES, rows - 1)) * p.n + min(j, p.n - 1)];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const unsigned long long bits = __ballot(b[u] != 0);
            if (i + u * WAVES < rows && lane < 2)
              seen_s[(i + u * WAVES) * kSeenPitch + (j - lane) / 32 + lane] = (uint32_t)(bits >> (32 * lane));
          }
        }
      __syncthreads();
    }
    // RW = 1: the tile's stage is filled again once it is read. RW > 1: after the
    // barrier that ends the wait for a tile, every wave has read the tile before it.
    const int turns = (nt + KG - 1) / KG;
    for (int i = 0, stage = 0; i < turns; ++i, stage = stage + 1 == NS ? 0 : stage + 1) {
      const int t = kg + i * KG;
      bits16* kt = ring + stage * 2 * T::ELEMS;
      if (RW == 1)
        wait_loads<(NS - 1) * 2 * LOADS>();
      else
        wait_loads<(NS - 2) * 2 * LOADS>();
      if (!all_in || k_begin + (t + 1) * T::KEYS > k_end) clear_tail(kt + T::ELEMS, t);
      if (RW > 1) {
        __syncthreads();
        issue(t + (NS - 1) * KG, stage == 0 ? NS - 1 : stage - 1);
      }
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int kb0 = k_begin + t * T::KEYS + st * 32;
        if (idle || kb0 >= k_end) continue;
        if (kb0 + 32 <= free_end)
          step(kt + st * 32 * N, kt + T::ELEMS + st * 32 * N, kb0, std::false_type{});
        else
          step(kt + st * 32 * N, kt + T::ELEMS + st * 32 * N, kb0, std::true_type{});
      }
      if (RW == 1) {
        wait_lds();
        issue(t + NS * KG, stage);
      }
    }
    wait_loads<0>();
    if (hidden) {  // wave-uniform: the masked steps' infinities and NaN
      for (int t = kg; t < nt; t += KG)
        for (int kb0 = k_begin + t * T::KEYS; kb0 < min(k_begin + (t + 1) * T::KEYS, k_end); kb0 += 32) {
          if (kb0 + 32 <= free_end) continue;
          const uint32_t seen = visible(kb0);
          // Bits of the lane's own half; the other half's keys come from lane ^ 32.
          const uint32_t other = __shfl_xor(seen, 32, 64), lo = h == 0 ? seen : other, hi = h == 0 ? other : seen;
#pragma unroll 1
          for (int i = 0; i < 32; ++i) {
            const int key = kb0 + i, b = (i >> 3) * 4 + (i & 3);
            const int page = key < k_end ? tab[(key >> cc.lg_page) - first] : -1;
            if (page < 0) continue;
            const bits16* row = cc.v + ((size_t)page * cc.Hkv + kv) * head_page + (size_t)(key & (cc.page - 1)) * N + 4 * h;
            const bool see = ((i & 4 ? hi : lo) >> b & 1) != 0;
#pragma unroll
            for (int db = 0; db < DB; ++db) add_not_finite<E>(o[db], row + 32 * db, see);
          }
        }
    }
  }

  if constexpr (KG > 1) {
    // The second key group's sums join the first's.
    f32x4* sx = reinterpret_cast<f32x4*>(smem_all) + (size_t)rw * DB * 4 * 64 + lane;
    const int me = rw * 64 + lane;
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          sx[(db * 4 + r4) * 64] = f32x4{o[db][4 * r4], o[db][4 * r4 + 1], o[db][4 * r4 + 2], o[db][4 * r4 + 3]};
      xm[me] = m_i;
      xl[me] = l_i;
    }
    __syncthreads();
    if (kg != 0) return;
    const float m1 = xm[me], m = fmaxf(m_i, m1);
    const float a0 = m_i == m ? 1.f : fast_exp2(m_i - m), a1 = m1 == m ? 1.f : fast_exp2(m1 - m);
    m_i = m;
    l_i = l_i * a0 + xl[me] * a1;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 x = sx[(db * 4 + r4) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[db][4 * r4 + e] = o[db][4 * r4 + e] * a0 + x[e] * a1;
      }
  }
  // Where the second launch finds the sequence's sums.
  if (p.part != nullptr && ck.chunk == 0 && kv == 0 && r0 == 0 && lane == 0) {
    int* head = reinterpret_cast<int*>(p.part) + 2 * s;
    head[0] = item;
    head[1] = ck.count;
  }
  const float l = l_i + __shfl_xor(l_i, 32, 64);
  if (r0 + c >= R) return;
  if (ck.count <= 1) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key: 0
    bits16* out = p.o + (((size_t)s * p.n + qi) * p.Hq + hq) * N + 4 * h;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x16& a = o[db];
        *reinterpret_cast<u32x2*>(out + 32 * db + 8 * r4) =
            u32x2{E::pack(a[4 * r4] * inv, a[4 * r4 + 1] * inv), E::pack(a[4 * r4 + 2] * inv, a[4 * r4 + 3] * inv)};
      }
    return;
  }
  float* part = p.part + tree_head_floats(cc.seqs) + (((size_t)item * cc.Hkv + kv) * R + r) * (N + 4);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x16& a = o[db];
      *reinterpret_cast<f32x4*>(part + 32 * db + 8 * r4 + 4 * h) = f32x4{a[4 * r4], a[4 * r4 + 1], a[4 * r4 + 2], a[4 * r4 + 3]};
    }
  if (h == 0) *reinterpret_cast<f32x4*>(part + N) = f32x4{m_i, l, 0.f, 0.f};
}

// o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a sequence's chunks, N / 4
// lanes a row. COOP, for few rows: one workgroup a row, 1024 / N chunks at a time,
// whose sums meet in LDS; else a row for each N / 4 lanes. Chunks without a key have
// m = -inf and l = 0; a row without any: 0.
template <class E, int N, bool COOP>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeParams p) {
  constexpr int L = N / 4, GR = 256 / L;
  __shared__ __attribute__((aligned(16))) float num_s[COOP ? GR : 1][COOP ? N : 4];
  __shared__ float den_s[GR], max_s[GR];
  const int G = p.Hq / p.c.Hkv, R = p.n * G, tid = threadIdx.x, gi = tid / L, d = tid % L * 4;
  const int s = blockIdx.x, row = COOP ? blockIdx.y : blockIdx.y * GR + gi;  // row: kv * R + r
  const int* head = reinterpret_cast<const int*>(p.part) + 2 * s;
  const int item = head[0], count = head[1];
  if (count <= 1 || row >= p.c.Hkv * R) return;  // written by the first launch (COOP: uniform)
  const size_t pitch = (size_t)p.c.Hkv * R * (N + 4);
  const float* part = p.part + tree_head_floats(p.c.seqs) + ((size_t)item * p.c.Hkv * R + row) * (N + 4);
  // Eight chunks at a time, all their loads in flight together; what was added so far
  // is scaled down where they have a larger maximum. (33 chunks of one token, the whole
  // call: 13.7 us; 15.3 with the maximum looked up first.)
  float M = -INFINITY, den = 0.f;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  constexpr int STEP = COOP ? GR : 1;
  for (int i0 = COOP ? gi : 0; i0 < count; i0 += 8 * STEP) {
    f32x4 ml[8], x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float* ps = part + (i0 + u * STEP) * pitch;
      ml[u] = f32x4{-INFINITY, 0.f, 0.f, 0.f};
      x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (i0 + u * STEP < count) {
        ml[u] = *reinterpret_cast<const f32x4*>(ps + N);
        x[u] = *reinterpret_cast<const f32x4*>(ps + d);
      }
    }
    float mx = M;
#pragma unroll
    for (int u = 0; u < 8; ++u) mx = fmaxf(mx, ml[u][0]);
    const float a = M == mx ? 1.f : exp2f(M - mx);
    num *= a;
    den *= a;
    M = mx;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      // (A chunk without weights holds zeros: its weight is made 0, not exp2(-inf + inf).)
      if (ml[u][1] == 0.f) continue;
      const float w = ml[u][0] == M ? 1.f : exp2f(ml[u][0] - M);
      den = __builtin_fmaf(w, ml[u][1], den);
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = __builtin_fmaf(w, x[u][e], num[e]);
    }
  }
  if (COOP) {
    *reinterpret_cast<f32x4*>(&num_s[gi][d]) = num;
    if (d == 0) {
      den_s[gi] = den;
      max_s[gi] = M;
    }
    __syncthreads();
    if (gi != 0) return;
    float mx = M;
#pragma unroll
    for (int g = 1; g < GR; ++g) mx = fmaxf(mx, max_s[g]);
    const float a = M == mx ? 1.f : exp2f(M - mx);
    num *= a;
    den *= a;
#pragma unroll
    for (int g = 1; g < GR; ++g) {
      const float b = max_s[g] == mx ? 1.f : exp2f(max_s[g] - mx);
      num += b * *reinterpret_cast<const f32x4*>(&num_s[g][d]);
      den = __builtin_fmaf(b, den_s[g], den);
    }
  }
  const float inv = den == 0.f ? 0.f : 1.0f / den;
  const int kv = row / R, r = row - kv * R, qi = r / G;
  *reinterpret_cast<u32x2*>(p.o + (((size_t)s * p.n + qi) * p.Hq + kv * G + (r - qi * G)) * N + d) =
      u32x2{E::pack(num[0] * inv, num[1] * inv), E::pack(num[2] * inv, num[3] * inv)};
}

template <class F>
void by_width(int N, F k) {
  if (N == 32) k(std::integral_constant<int, 32>{});
  if (N == 64) k(std::integral_constant<int, 64>{});
  if (N == 128) k(std::integral_constant<int, 128>{});
  if (N == 256) k(std::integral_constant<int, 256>{});
}

template <class E>
hipError_t launch_tree(const TreeParams& p, hipStream_t s) {
  by_width(p.c.N, [&](auto n) {
    constexpr int N = decltype(n)::value;
    const TreeGrid g = tree_grid(p.c.seqs, p.c.Hkv, p.n * (p.Hq / p.c.Hkv), p.c.max_pages << p.c.lg_page, N);
    const dim3 grid((unsigned)(g.items * g.row_groups * p.c.Hkv));
    if (g.blocks == 1)
      hipLaunchKernelGGL((tree_attn_kernel<E, N, 1>), grid, dim3((64 * Tile<N, 1>::WAVES)), 0, s, p);
    else if (g.blocks == 2)
      hipLaunchKernelGGL((tree_attn_kernel<E, N, 2>), grid, dim3((64 * Tile<N, 2>::WAVES)), 0, s, p);
    else
      hipLaunchKernelGGL((tree_attn_kernel<E, N, 4>), grid, dim3((64 * Tile<N, 4>::WAVES)), 0, s, p);
  });
  return hipGetLastError();
}

template <class E>
hipError_t launch_combine(const TreeParams& p, hipStream_t s) {
  const int rows = p.n * p.Hq;
  by_width(p.c.N, [&](auto n) {
    constexpr int N = decltype(n)::value, GR = 1024 / N;
    // A workgroup a row while that leaves them few (N = 128; 1024 rows of 64 chunks:
    // 9.3 us so, 27 with a row for each 32 lanes; 8192 rows of 8 chunks: 24 / 11).
    if ((int64_t)p.c.seqs * rows <= 2048)
      hipLaunchKernelGGL((tree_combine_kernel<E, N, true>), dim3(p.c.seqs, rows), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((tree_combine_kernel<E, N, false>), dim3(p.c.seqs, (rows + GR - 1) / GR), dim3(256), 0, s, p);
  });
  return hipGetLastError();
}

template <int N>
int turn_of(int blocks) {
  return blocks == 1 ? Tile<N, 1>::TURN : blocks == 2 ? Tile<N, 2>::TURN : Tile<N, 4>::TURN;
}
template <int N>
int slots_of(int blocks) {
  return blocks == 1 ? Tile<N, 1>::SLOTS : blocks == 2 ? Tile<N, 2>::SLOTS : Tile<N, 4>::SLOTS;
}

}  // namespace

// blocks: waves of 32 query rows that share a workgroup's tiles; want: chunks of a
// head that run at one time (0: chunks of the largest size); items: a bound of a
// head's chunks.
TreeGrid tree_grid(int seqs, int Hkv, int rows, int capacity, int N) {
  TreeGrid g;
  const int need = (rows + 31) / 32;
  g.blocks = need <= 2 ? need : 4;
  g.row_groups = (need + g.blocks - 1) / g.blocks;
  g.turn = N == 32 ? turn_of<32>(g.blocks) : N == 64 ? turn_of<64>(g.blocks) : N == 128 ? turn_of<128>(g.blocks) : turn_of<256>(g.blocks);
  const int64_t lanes = (int64_t)Hkv * g.row_groups;
  const int slots = N == 32 ? slots_of<32>(g.blocks) : N == 64 ? slots_of<64>(g.blocks) : N == 128 ? slots_of<128>(g.blocks) : slots_of<256>(g.blocks);
  g.full = (capacity + kMaxChunk - 1) / kMaxChunk;
  const int64_t full = (int64_t)seqs * g.full;
  if (seqs > kManySeqs || (int64_t)seqs * (capacity / 16 + 1) >= INT64_C(1) << 31) {
    g.want = 0;
    g.least = kMaxChunk;
    g.items = full;
    g.split = capacity > kMaxChunk;
    return g;
  }
  // Few sequences: at most `want` chunks, many: 4 * want and one for each; or the
  // largest chunks, if they are more; no more than the capacity has of the smallest.
  g.want = (int)(slots / lanes > 1 ? slots / lanes : 1);
  // Keys of a chunk at least. Many sequences: what a workgroup's start and the sums' way
  // through memory are worth (64 sequences of up to 1024 rows of 8 heads, one token:
  // chunks of 150 keys 61 us, whole sequences 48; of up to 2048: 90 and 82). Few: two
  // turns, or one where its sums are small beside its keys (N = 128, one sequence of
  // 4096 rows, 4 query rows a head: 13.6 us with two, 13.1 with one; 64: 16.4 and 19.0).
  const bool few = 2 * seqs <= g.want;
  g.least = !few ? kLeast : 4 * rows <= g.turn ? g.turn : 2 * g.turn;
  const int64_t most = (int64_t)seqs * ((capacity + g.least - 1) / g.least);
  g.items = few ? g.want : 4 * g.want + seqs;
  if (g.items < full) g.items = full;
  if (g.items > most) g.items = most;
  g.split = capacity > g.least;
  return g;
}

hipError_t launch_tree_attn(const TreeParams& p, bool fp16, hipStream_t s) {
  return fp16 ? launch_tree<Fp16>(p, s) : launch_tree<Bf16>(p, s);
}
hipError_t launch_tree_combine(const TreeParams& p, bool fp16, hipStream_t s) {
  return fp16 ? launch_combine<Fp16>(p, s) : launch_combine<Bf16>(p, s);
}

}  // namespace mea
