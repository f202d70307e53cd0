// Attention of n new tokens per sequence over a paged cache on gfx950 MFMA: one
// token of a decoding step (n = 1), or a drafted tree whose tokens see their
// ancestors. The new tokens' k and v are already the last n rows of the cache:
//   o_i = sum_r w_ir v_r / sum_r w_ir,  w_ir = exp(scale q_i . k_r)  over the rows
//   r < len - n, and r = len - n + j where mask[i][j];  0 where there is none.
//
// Bound by reading the cache once from HBM: the rows of a key head are read for
// all its R = n * G query rows together (row i * G + g, G query heads to a key
// head), 32 of them to a block of v_mfma_f32_32x32x16, the query on the lane (the
// forms of attn_fwd.hip, S^T = K Q^T, O^T += V^T P^T). A workgroup's four waves
// are RW blocks of query rows times KG groups of keys; a tile of 32 * KG * ST keys
// streams into LDS double-buffered and key group kg takes its own ST * 32. Few
// query rows leave the keys to be split (flash decoding): over the key groups,
// whose sums meet in LDS, and over `splits` workgroups of whole tiles, whose
// fp32 sums the second launch adds in order.
//
// Pages: the split's table entries are read once into LDS; each lane of a tile
// load finds its own row's page there. Rows past the sequence and rows of pages
// outside the pool read the pool's first row and are masked.
#include <type_traits>

#include "elem.cuh"
#include "grouped.h"

namespace mea {

namespace {

// Tile geometry by head width and query blocks per workgroup.
template <int N, int RW>
struct Shape {
  static constexpr int KG = N == 256 ? 2 : 4 / RW;  // key groups
  static constexpr int ST = RW == 4 ? 2 : 1;        // 32-key steps of a group per tile
  static constexpr int WAVES = RW * KG, BK = 32 * KG * ST;
};
constexpr int kMaxSplitKeys = 8192;                  // keys of a split
constexpr int kTab = kMaxSplitKeys / 16 + 2;         // its table entries at 16 rows a page

template <class E, int N, int RW>
__global__ __launch_bounds__((64 * Shape<N, RW>::WAVES), 1) void tree_attn_kernel(TreeParams p) {
  using S = Shape<N, RW>;
  constexpr int KG = S::KG, ST = S::ST, WAVES = S::WAVES, BK = S::BK;
  constexpr int CH = N / 8, KS = N / 16, DB = N / 32;
  constexpr int TILE = BK * N;
  constexpr int LOADS = TILE / 8 / (64 * WAVES);
  constexpr int XCH = KG > 1 ? RW * DB * 16 * 64 * 2 : 0;  // one group's fp32 sums (16-bit elements)
  constexpr int SMEM = 4 * TILE > XCH ? 4 * TILE : XCH;
  __shared__ __attribute__((aligned(16))) bits16 smem[SMEM];  // [stage][K | V], then the exchange
  __shared__ int tab[kTab];
  __shared__ float xm[KG > 1 ? RW * 64 : 1], xl[KG > 1 ? RW * 64 : 1];

  const PagedCache& cc = p.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave % RW, kg = wave / RW;
  const int c = lane & 31, h = lane >> 5;
  const int G = p.Hq / cc.Hkv, R = p.n * G;
  const int kv = blockIdx.x % cc.Hkv, s = blockIdx.x / cc.Hkv, split = blockIdx.y;
  const int r0 = (blockIdx.z * RW + rw) * 32;  // this wave's query rows
  const int len = __builtin_amdgcn_readfirstlane(min(max(cc.lengths[s], 0), cc.max_pages << cc.lg_page));
  const int ctx = max(len - p.n, 0), lead = p.n - (len - ctx);  // lead: tokens in front of an empty sequence's rows
  // Whole tiles per split.
  const int per = (len + p.splits * BK - 1) / (p.splits * BK) * BK;
  const int k_begin = split * per, k_end = min(k_begin + per, len);

  // Query row r = i * G + g: token i, head kv * G + g.
  const int r = min(r0 + c, R - 1), qi = r / G;
  const size_t hq = (size_t)kv * G + (r - qi * G);

  float m_i = -INFINITY, l_i = 0.f;  // l_i: this lane's half of the keys
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();

  if (k_begin < k_end) {  // uniform over the workgroup
    // Table entries of the split; whether all of them lie in the pool.
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
    const uint32_t smem_b = lds_addr(smem);
    auto issue_tile = [&](int j0, int stage) {
      const uint32_t at = smem_b + (uint32_t)(stage * 2 * TILE) * 2u;
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int slot = (u * WAVES + wave) * 64 + lane;
        const int row = slot / CH, key = j0 + row;
        const int page = key < k_end ? tab[(key >> cc.lg_page) - first] : -1;
        const size_t off = (page < 0 ? 0 : ((size_t)page * cc.Hkv + kv) * head_page + (size_t)(key & (cc.page - 1)) * N) +
                           ((slot % CH) ^ chunk_swz<CH>(row)) * 8;
        g2lds16(cc.k + off, at + (uint32_t)(u * WAVES + wave) * 1024u);
        g2lds16(cc.v + off, at + TILE * 2u + (uint32_t)(u * WAVES + wave) * 1024u);
      }
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

    // Whether this lane's query sees row `key`.
    const unsigned char* mrow = p.mask == nullptr ? nullptr : p.mask + s * p.mask_seq + (int64_t)qi * p.n;
    auto sees = [&](int key) {
      if (key >= k_end || tab[(key >> cc.lg_page) - first] < 0) return false;
      if (key < ctx) return true;
      const int j = key - ctx + lead;  // token of the row
      return mrow == nullptr ? j <= qi : mrow[j] != 0;
    };

    // One 32-key step, as in the forward of the packed prompts; MASK: some row may
    // be hidden from some query. A query that has seen no key yet has m = -inf.
    int hidden = 0;  // masked steps whose V holds infinities or NaN, left out there
    auto step = [&](const bits16* kt, const bits16* vt, int kb0, auto mask_tag) {
      constexpr bool MASK = decltype(mask_tag)::value;
      uint32_t seen = 0xFFFFu;
      if (MASK) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) seen |= (uint32_t)sees(kb0 + 8 * (i >> 2) + 4 * h + (i & 3)) << i;
      }
      f32x16 w = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) w = E::mma(*reinterpret_cast<const u32x4*>(kt + koff[ks]), qf[ks], w);
      if (MASK) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((seen >> i & 1) == 0) w[i] = -INFINITY;
      }
      const f32x16 sc = w;
      float top_w;
      auto weigh = [&](float m) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = fast_exp2(__builtin_fmaf(sc[i], p.sl2e, -m));
        top_w = w[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top_w = fmaxf(top_w, w[i]);
      };
      weigh(m_i);
      const bool over = !(top_w <= E::kMaxWeight);
      if (__any(over)) {
        const bool up = ((int)over | __shfl_xor((int)over, 32, 64)) != 0;  // (every lane takes part in the exchange)
        float mx = sc[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = up ? fmaxf(m_i, mx * p.sl2e) : m_i;
        const float a = mn == m_i ? 1.f : fast_exp2(m_i - mn);
        l_i *= a;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= a;
        m_i = mn;
        // No key seen: weights exp2(-inf - 0) = 0. (NaN scores stay NaN.)
        weigh(m_i == -INFINITY ? 0.f : m_i);
      }
      u32x4 pf[2];
#pragma unroll
      for (int kst = 0; kst < 2; ++kst)
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[kst][e] = E::pack(w[8 * kst + 2 * e], w[8 * kst + 2 * e + 1]);
      l_i = E::add_weights(l_i, w, pf);
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
          hidden = 1;
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

    const int nt = (k_end - k_begin + BK - 1) / BK;
    // Rows that every query sees: whole steps below free_end.
    const int free_end = all_in ? min(ctx, k_end) : 0;
    const bool idle = r0 >= R;  // no query rows left for this wave
    issue_tile(k_begin, 0);
    wait_vmcnt0();
    __syncthreads();
    for (int j = 0; j < nt; ++j) {
      const int j0 = k_begin + j * BK;
      if (j + 1 < nt) issue_tile(j0 + BK, (j + 1) & 1);
      const bits16* kt = smem + (j & 1) * 2 * TILE;
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int row = (kg * ST + st) * 32, kb0 = j0 + row;
        if (idle || kb0 >= k_end) continue;
        if (kb0 + 32 <= free_end)
          step(kt + row * N, kt + TILE + row * N, kb0, std::false_type{});
        else
          step(kt + row * N, kt + TILE + row * N, kb0, std::true_type{});
      }
      wait_vmcnt0();
      __syncthreads();
    }
    if (hidden) {  // wave-uniform: the masked steps' infinities and NaN
      for (int j = 0; j < nt; ++j)
        for (int st = 0; st < ST; ++st) {
          const int kb0 = k_begin + j * BK + (kg * ST + st) * 32;
          if (kb0 >= k_end || kb0 + 32 <= free_end) continue;
          for (int key = kb0; key < min(kb0 + 32, k_end); ++key) {
            const int page = tab[(key >> cc.lg_page) - first];
            if (page < 0) continue;
            const bits16* row = cc.v + ((size_t)page * cc.Hkv + kv) * head_page + (size_t)(key & (cc.page - 1)) * N + 4 * h;
            const bool see = sees(key);
#pragma unroll
            for (int db = 0; db < DB; ++db) add_not_finite<E>(o[db], row + 32 * db, see);
          }
        }
    }
  }

  if constexpr (KG > 1) {
    // The key groups' sums join group 0's, one group after the other.
    f32x4* sx = reinterpret_cast<f32x4*>(smem) + (size_t)rw * DB * 4 * 64 + lane;
    const int me = rw * 64 + lane;
    for (int from = 1; from < KG; ++from) {
      if (kg == from) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4)
            sx[(db * 4 + r4) * 64] = f32x4{o[db][4 * r4], o[db][4 * r4 + 1], o[db][4 * r4 + 2], o[db][4 * r4 + 3]};
        xm[me] = m_i;
        xl[me] = l_i;
      }
      __syncthreads();
      if (kg == 0) {
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
      __syncthreads();
    }
    if (kg != 0) return;
  }
  if (r0 + c >= R) return;
  const float l = l_i + __shfl_xor(l_i, 32, 64);
  if (p.splits == 1) {
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
  float* part = p.part + (((size_t)blockIdx.x * p.splits + split) * R + r) * (N + 4);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x16& a = o[db];
      *reinterpret_cast<f32x4*>(part + 32 * db + 8 * r4 + 4 * h) = f32x4{a[4 * r4], a[4 * r4 + 1], a[4 * r4 + 2], a[4 * r4 + 3]};
    }
  if (h == 0) *reinterpret_cast<f32x4*>(part + N) = f32x4{m_i, l, 0.f, 0.f};
}

// o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the splits, N / 4 lanes per
// query row. Splits without a key have m = -inf and l = 0; a row without any: 0.
template <class E, int N>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeParams p) {
  constexpr int L = N / 4;  // lanes per row
  const int G = p.Hq / p.c.Hkv, R = p.n * G;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / L;
  if (row >= (int64_t)p.c.seqs * p.c.Hkv * R) return;
  const int d = (int)(id % L) * 4;
  const int64_t bh = row / R;
  const int r = (int)(row - bh * R), s = (int)(bh / p.c.Hkv), kv = (int)(bh - (int64_t)s * p.c.Hkv);
  const float* part = p.part + ((size_t)bh * p.splits * R + r) * (N + 4);
  const size_t pitch = (size_t)R * (N + 4);
  float M = -INFINITY;
  for (int i = 0; i < p.splits; ++i) M = fmaxf(M, part[i * pitch + N]);
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  for (int i = 0; i < p.splits; ++i) {
    const float* ps = part + i * pitch;
    const float m = ps[N], w = m == M ? 1.f : exp2f(m - M);
    const f32x4 x = *reinterpret_cast<const f32x4*>(ps + d);
    if (ps[N + 1] == 0.f) continue;  // (0 weights and no keys: nothing to add)
    den = __builtin_fmaf(w, ps[N + 1], den);
#pragma unroll
    for (int e = 0; e < 4; ++e) num[e] = __builtin_fmaf(w, x[e], num[e]);
  }
  const float inv = den == 0.f ? 0.f : 1.0f / den;
  const int qi = r / G;
  *reinterpret_cast<u32x2*>(p.o + (((size_t)s * p.n + qi) * p.Hq + kv * G + (r - qi * G)) * N + d) =
      u32x2{E::pack(num[0] * inv, num[1] * inv), E::pack(num[2] * inv, num[3] * inv)};
}

template <class E, int N>
void launch_tree(const TreeParams& p, hipStream_t s) {
  const int R = p.n * (p.Hq / p.c.Hkv), blocks = (R + 31) / 32;
  const dim3 grid(p.c.seqs * p.c.Hkv, p.splits);
  auto go = [&](auto rw) {
    constexpr int RW = decltype(rw)::value;
    hipLaunchKernelGGL((tree_attn_kernel<E, N, RW>), dim3(grid.x, grid.y, (blocks + RW - 1) / RW),
                       dim3(64 * Shape<N, RW>::WAVES), 0, s, p);
  };
  if (blocks == 1)
    go(std::integral_constant<int, 1>{});
  else if (blocks == 2 || N == 256)
    go(std::integral_constant<int, 2>{});
  else if constexpr (N < 256)
    go(std::integral_constant<int, 4>{});
}

template <class E>
hipError_t launch_tree_n(const TreeParams& p, hipStream_t s) {
  switch (p.c.N) {
    case 32: launch_tree<E, 32>(p, s); break;
    case 64: launch_tree<E, 64>(p, s); break;
    case 128: launch_tree<E, 128>(p, s); break;
    case 256: launch_tree<E, 256>(p, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <class E>
hipError_t launch_combine_n(const TreeParams& p, hipStream_t s) {
  const int64_t rows = (int64_t)p.c.seqs * p.n * p.Hq;
  const dim3 grid((unsigned)((rows * (p.c.N / 4) + 255) / 256));
  switch (p.c.N) {
    case 32: hipLaunchKernelGGL((tree_combine_kernel<E, 32>), grid, dim3(256), 0, s, p); break;
    case 64: hipLaunchKernelGGL((tree_combine_kernel<E, 64>), grid, dim3(256), 0, s, p); break;
    case 128: hipLaunchKernelGGL((tree_combine_kernel<E, 128>), grid, dim3(256), 0, s, p); break;
    case 256: hipLaunchKernelGGL((tree_combine_kernel<E, 256>), grid, dim3(256), 0, s, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

// Splits of a sequence's keys: as many workgroups as fill the card twice, as far
// as the capacity gives each two tiles; and enough that a split's table fits LDS.
int tree_splits(int seqs, int Hkv, int rows, int capacity, int N) {
  const int blocks = (rows + 31) / 32, rw = blocks == 1 ? 1 : blocks == 2 || N == 256 ? 2 : 4;
  const int bk = N == 256 ? 64 : rw == 1 ? 128 : 64;
  const int64_t wgs = (int64_t)seqs * Hkv * ((blocks + rw - 1) / rw);
  const int64_t tiles = (capacity + bk - 1) / bk;
  int64_t s = (512 + wgs - 1) / wgs;
  if (s > (tiles + 1) / 2) s = (tiles + 1) / 2;
  const int64_t least = (capacity + kMaxSplitKeys - bk - 1) / (kMaxSplitKeys - bk);
  if (s < least) s = least;
  return s < 1 ? 1 : (int)s;
}

hipError_t launch_tree_attn(const TreeParams& p, bool fp16, hipStream_t s) {
  return fp16 ? launch_tree_n<Fp16>(p, s) : launch_tree_n<Bf16>(p, s);
}
hipError_t launch_tree_combine(const TreeParams& p, bool fp16, hipStream_t s) {
  return fp16 ? launch_combine_n<Fp16>(p, s) : launch_combine_n<Bf16>(p, s);
}

}  // namespace mea
