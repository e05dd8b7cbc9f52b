// Single-query attention of a batch that shares a prefix (gfx950): every
// sequence attends the prefix's pages and then its own.
//
//   o_b = softmax(scale q_b [K_prefix; K_b]^T) [V_prefix; V_b]
//
// A paged decode reads the prefix once per sequence. Here the B g query rows
// of a KV head (all sequences, g heads each) are one matrix against it. Two
// launches:
//  * pf_prefix_kernel: one workgroup per work item. A prefix item is 128 rows
//    of a KV head against one chunk of the prefix's keys; an own item is the g
//    rows of one sequence and KV head against one chunk of the sequence's keys.
//    Each leaves (max, sum, acc) of its rows in float32. The prefix items come
//    first: they are bound by the matrix cores where there are many sequences,
//    the own items by memory, and both kinds then run beside each other.
//  * pf_prefix_merge_kernel: o = sum_i acc_i 2^(m_i - M) / sum_i l_i 2^(m_i - M)
//    over a row's chunks.
// No counterpart in the reference, whose paged call gives the prefix's pages
// to every sequence's table (paged.py:102-192).
//
// An item runs the prefill forward's pipeline (attn_fwd.hip) over pages: K one
// 64-key block ahead of V, both double-buffered in LDS; S^T = K Q^T runs beside
// the exponentials of the block before, O^T += V^T P^T beside the maximum of the
// block after. The tiles come by direct global -> LDS loads of whole rows (1 KB
// each, inside one page; rows past the length and columns past the stored head
// dim lie outside the load's buffer range and arrive as zeros). The pages' first
// rows are looked up once, into LDS. Pages that such loads would straddle and
// unaligned pools are staged through registers instead.
#include "pf_common.hpp"
#include "pf_kernels.hpp"
#include "pf_tiles.hpp"

namespace pf {

namespace {

constexpr int kBN = 64;      // keys per block
constexpr int kRows = kPrefixRows;

// Scalar load of a wave-uniform address.
__device__ inline int sload(const int32_t* a) {
  const __attribute__((address_space(4))) int32_t* c = (const __attribute__((address_space(4))) int32_t*)a;
  return __builtin_amdgcn_readfirstlane(*c);
}
// Keys of the prefix, and of sequence b on its own.
__device__ inline int prefix_len(const PrefixParams& p) {
  return p.len_ptr != nullptr ? min(max(sload(p.len_ptr), 0), p.len) : p.len;
}
__device__ inline int own_len(const PrefixParams& p, int b) { return min(max(sload(p.own_lens + b), 0), p.own_cap); }

// Loads of 64-row tiles of keys [key0, key0 + kv_len) of a table's pages. DMA:
// each wave's loads are RPL whole rows of one page; else every lane fetches its
// 16-byte chunks itself.
template <typename T, int D, bool DMA>
struct PageTiles {
  using G = Tile<T, D>;
  static constexpr int PT = G::CPR / 4;         // loads per lane and tile
  static constexpr int RPL = 1024 / G::RB;      // rows per load
  uint32_t voff[PT];  // DMA: the lane's byte offset within the load's rows
  uint32_t row0;      // DMA: the wave's first row of load 0; load u: + 4 RPL u
  uint32_t slot0;     // the wave's LDS byte offset of load 0; load u: + 4096 u
  int lane, kv_len, last, key0, kvh;
  const PrefixParams& p;
  const int32_t* table;
  const uint32_t* first;  // LDS: pool row of each group of keys

  // groups: of keys looked up, at least 1
  __device__ inline PageTiles(const PrefixParams& p_, int tid, int key0_, int kv_len_, int groups, int kvh_,
                              const int32_t* table_, const uint32_t* first_)
      : lane(tid & 63), kv_len(kv_len_), last(groups - 1), key0(key0_), kvh(kvh_), p(p_), table(table_), first(first_) {
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    row0 = RPL * w;
    slot0 = 1024 * w;
#pragma unroll
    for (int u = 0; u < PT; ++u) {
      const int r = lane / G::CPR, row = RPL * (4 * u + w) + r;
      const int chunk = (lane % G::CPR) ^ tile_swz<G::CPR>(row);
      // columns past the stored row: past any range
      voff[u] = chunk * G::EPC < p.dr ? (uint32_t)((r * p.dr + chunk * G::EPC) * G::ES) : 0x7ffffff0u;
    }
  }
  // The pool row of load u of block j.
  __device__ inline uint32_t row_of(int j, int u) const {
    const int key = kBN * j + row0 + 4 * RPL * u;
    const int grp = min(key >> p.group_log2, last);
    return __builtin_amdgcn_readfirstlane(first[grp]) + (key & ((1 << p.group_log2) - 1));
  }
  __device__ inline void load(const void* pool, uint32_t row, int j, int u, char* tile) const {
    const int key = kBN * j + row0 + 4 * RPL * u;
    const int valid = min(max(kv_len - key, 0), RPL);
    const uint32_t rb = p.dr * G::ES;
    const i32x4 d = make_desc(static_cast<const char*>(pool) + (uint64_t)row * rb, valid * rb);
    dma16(d, voff[u], __builtin_amdgcn_readfirstlane(lds_u32(tile) + slot0 + 4096 * u));
  }
  // Without DMA: block j through registers.
  __device__ inline void copy(const void* pool, int j, char* tile) const {
    u32x4 x[PT];
#pragma unroll
    for (int u = 0; u < PT; ++u) {
      const int s = (slot0 + 4096 * u) / 16 + lane, row = s / G::CPR;
      const int chunk = (s % G::CPR) ^ tile_swz<G::CPR>(row), key = kBN * j + row;
      x[u] = (u32x4){0u, 0u, 0u, 0u};
      if (key < kv_len && chunk * G::EPC < p.dr) {
        const int lp = (key0 + key) / p.page_size;
        const int page = min(max(table[lp], 0), p.num_pages - 1);
        const int64_t at = ((int64_t)page * p.Hkv + kvh) * p.page_size + (key0 + key - lp * p.page_size);
        x[u] = ldg16(static_cast<const T*>(pool) + at * p.dr + chunk * G::EPC);
      }
    }
#pragma unroll
    for (int u = 0; u < PT; ++u) sts16(tile + slot0 + 4096 * u + 16 * lane, x[u]);
  }
};

template <typename T, int D, bool DMA>
__global__ __launch_bounds__(256, (kFwdWgPerCu<T, D>)) void pf_prefix_kernel(PrefixParams p) {
  using MF = Mfma32<T>;
  using Frag = typename MF::Frag;
  using G = Tile<T, D>;
  using PTiles = PageTiles<T, D, DMA>;
  constexpr int HALF = D / 2, EPC = G::EPC, FPC = frags_per_chunk<T>();
  constexpr int QF = HALF / MF::kK, NDT = D / 32, PF = 32 / MF::kK, PT = PTiles::PT;
  __shared__ __attribute__((aligned(1024))) char smem[4 * G::BYTES];  // K blocks j & 1, then V blocks
  __shared__ uint32_t first[DMA ? kPrefixGroups : 1];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hh = lane >> 5, l32 = lane & 31;

  // The item: rows, table, and keys [key0, key0 + chunk) below len.
  const int32_t* table;
  int kvh, b0, r0, piece, key0, chunk, cap, len;
  const bool own = blockIdx.x >= (unsigned)p.n_pre;
  if (!own) {
    // (chunk, kv head, row tile): the row tiles of one chunk side by side on one
    // XCD, whose L2 then serves the chunk to all of them.
    const int item = xcd_remap(blockIdx.x, p.n_pre, p.n_tiles);
    r0 = kRows * (item % p.n_tiles);
    kvh = item / p.n_tiles % p.Hkv;
    piece = item / p.n_tiles / p.Hkv;
    b0 = 0;
    table = p.table;
    chunk = p.chunk;
    key0 = piece * chunk;
    cap = p.len;
    len = prefix_len(p);
  } else {
    // chunk by chunk, so that the items past the sequences' ends come last
    const int item = blockIdx.x - p.n_pre, seqs = p.B * p.Hkv * p.n_hc;
    const int c = item / seqs, sq = item - c * seqs;
    r0 = kRows * (sq % p.n_hc);
    kvh = sq / p.n_hc % p.Hkv;
    b0 = sq / p.n_hc / p.Hkv;
    piece = p.n_split + c;
    table = p.own_tables + (int64_t)b0 * p.pages_per_seq;
    chunk = p.own_chunk;
    key0 = c * chunk;
    cap = p.own_cap;
    len = own_len(p, b0);
  }
  // The lookups do not wait for the length: entries past it (-1 padding) are
  // clamped, and no row of theirs is read.
  const int groups = (min(chunk, cap - key0) + (1 << p.group_log2) - 1) >> p.group_log2;
  if constexpr (DMA) {
    for (int i = tid; i < groups; i += 256) {
      const int key = key0 + (i << p.group_log2);
      const int lp = key / p.page_size;
      const int page = min(max(table[lp], 0), p.num_pages - 1);
      first[i] = ((uint32_t)page * p.Hkv + kvh) * p.page_size + (key - lp * p.page_size);
    }
  }
  if (key0 >= len) return;  // the merge counts the chunks below len
  const int kv_len = min(len - key0, chunk);
  const int nblk = (kv_len + kBN - 1) / kBN;
  if constexpr (DMA) __syncthreads();
  const PTiles tiles(p, tid, key0, kv_len, groups, kvh, table, first);
  char* const kbuf0 = smem;
  char* const vbuf0 = smem + 2 * G::BYTES;
  auto whole = [&](const void* pool, int j, char* t) {
    if constexpr (DMA) {
#pragma unroll
      for (int u = 0; u < PT; ++u) tiles.load(pool, tiles.row_of(j, u), j, u, t);
    } else {
      tiles.copy(pool, j, t);
    }
  };
  whole(p.k, 0, kbuf0);
  whole(p.v, 0, vbuf0);
  if (nblk > 1) whole(p.k, 1, kbuf0 + G::BYTES);

  // Q: the lane's row, columns [hh HALF, + HALF). An own item seldom has rows for
  // more than one wave: which one differs from item to item, so that the items
  // on a CU load all of its SIMDs.
  const int rw = r0 + 32 * (own ? (wv + blockIdx.x) & 3 : wv), r = rw + l32;
  const int n_rows = own ? p.g : p.rows;
  const bool active = rw < n_rows;  // the wave has rows at all
  const int b = own ? b0 : r / p.g, h = kvh * p.g + (own ? r : r - b * p.g);
  Frag qf[QF];
  {
    const T* qr = static_cast<const T*>(p.q) + ((int64_t)b * p.Hq + h) * p.dr + hh * HALF;
    u32x4 qc[HALF / EPC];
#pragma unroll
    for (int c = 0; c < HALF / EPC; ++c)
      qc[c] = r < n_rows && hh * HALF + c * EPC < p.dr ? ldg16(qr + c * EPC) : (u32x4){0u, 0u, 0u, 0u};
    if (p.scale_log2 < 0.f) {  // |scale| on -Q
      const uint32_t sign = G::ES == 4 ? 0x80000000u : 0x80008000u;
#pragma unroll
      for (int c = 0; c < HALF / EPC; ++c) qc[c] ^= (u32x4){sign, sign, sign, sign};
    }
#pragma unroll
    for (int c = 0; c < HALF / EPC; ++c)
#pragma unroll
      for (int f = 0; f < FPC; ++f) qf[c * FPC + f] = chunk_frag<T>(qc[c], f);
  }

  // Running maximum (log2 units) from the lowest finite value: scores of -inf
  // weigh nothing and a row of nothing else keeps sum 0.
  float m_run = -__FLT_MAX__, l_run = 0.f;
  f32x16 acc[NDT];
#pragma unroll
  for (int i = 0; i < NDT; ++i) acc[i] = (f32x16)(0.f);
  const float c2 = fmaxf(fabsf(p.scale_log2), 1e-30f);  // masked scores (-inf) stay -inf
  TrAddr<T, D> vta;
  vta.init(lane);

  // m_run moves when some row's maximum grows by more than 8: p <= 2^8, and the
  // rescaling is rare.
  auto update_max = [&](float mx) {
    const float m_cand = fmaxf(m_run, mx);
    if (__any(m_cand > m_run + 8.f)) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_cand);
#pragma unroll
      for (int i = 0; i < NDT; ++i) acc[i] *= alpha;
      l_run *= alpha;
      m_run = m_cand;
    }
  };
  // The lane's maximum of a block's scores; keys at or past kv_len become -inf.
  auto block_max = [&](f32x16* s, int kv0) {
    const int rel = kv_len - kv0 - 32 * hh;
    float mx = kNegInf;
#pragma unroll
    for (int v = 0; v < 32; ++v) {
      const float x = v < rel ? s[v >> 4][v & 15] : kNegInf;
      s[v >> 4][v & 15] = x;
      mx = fmaxf(mx, x);
    }
    return mx;
  };

  dma_wait();
  __syncthreads();
  f32x16 s_cur[2] = {(f32x16)(0.f), (f32x16)(0.f)};
  float mx_carry = kNegInf;  // the lane's maximum of the latest block, not yet applied
  if (active) {
    mfma_nat<T, D>(kbuf0, l32, hh, qf, s_cur[0], s_cur[1]);
    mx_carry = block_max(s_cur, 0);
  }
  __syncthreads();  // K_0 is read before K_2 overwrites it

  uint32_t row_k[PT], row_v[PT];  // DMA: pool rows of the loads of K_{j+2} and V_{j+1}
  if constexpr (DMA) {
#pragma unroll
    for (int u = 0; u < PT; ++u) row_v[u] = tiles.row_of(1, u);
  }
  for (int j = 0; j + 1 < nblk; ++j) {
    char* const kcur = kbuf0 + ((j + 1) & 1) * G::BYTES;  // K_{j+1}
    char* const vcur = vbuf0 + (j & 1) * G::BYTES;        // V_j
    char* const kdst = kbuf0 + (j & 1) * G::BYTES;        // K_{j+2}
    char* const vdst = vbuf0 + ((j + 1) & 1) * G::BYTES;  // V_{j+1}
    const bool k_next = j + 2 < nblk;
    auto load_part = [&](int i) __attribute__((always_inline)) {
      if constexpr (DMA) {
        if (i < PT) {
          if (k_next) tiles.load(p.k, row_k[i], j + 2, i, kdst);
        } else if (i < 2 * PT) {
          tiles.load(p.v, row_v[i - PT], j + 1, i - PT, vdst);
        }
      }
    };
    if constexpr (DMA) {
#pragma unroll
      for (int u = 0; u < PT; ++u) row_k[u] = tiles.row_of(j + 2, u);
    } else {
      if (k_next) tiles.copy(p.k, j + 2, kdst);
      tiles.copy(p.v, j + 1, vdst);
    }
    if (!active) {
#pragma unroll
      for (int i = 0; i < 2 * PT; ++i) load_part(i);
    } else {
      f32x16 s_nxt[2] = {(f32x16)(0.f), (f32x16)(0.f)};
      Frag pfr[PF];
      const bool masked = (j + 2) * kBN > kv_len;
      if constexpr (sizeof(T) == 2) {
        // As in the forward: S_{j+1} beside the maximum and the first quarter of
        // S_j's exponentials, P.V beside the rest.
        constexpr int NV1 = G::CPR, NV2 = 4 * NDT, VPS2 = 32 / NV2;
        uint32_t pw[16];
        float rs = 0.f, mxr = kNegInf, mx = kNegInf;
        auto exp_pair = [&](int pr) __attribute__((always_inline)) {
          const int v = 2 * pr;
          const float x0 = __builtin_amdgcn_exp2f(fmaf(s_cur[v >> 4][v & 15], c2, -m_run));
          const float x1 = __builtin_amdgcn_exp2f(fmaf(s_cur[v >> 4][(v & 15) + 1], c2, -m_run));
          pw[pr] = pack2<T>(x0, x1);
          rs += x0 + x1;  // the sum is of the unrounded weights
          asm volatile("" : "+v"(rs));  // keeps the sum beside its MFMA
        };
        mfma_nat_il<T, D>(kcur, l32, hh, qf, s_nxt[0], s_nxt[1], [&](int i) {
          load_part(i);
          if (i == 0) {
            mxr = wave_xor32_max(mx_carry) * c2;
          } else if (i == 1) {
            update_max(mxr);
          } else {
#pragma unroll
            for (int pr = ((i - 2) * 4) / (NV1 - 2); pr < ((i - 1) * 4) / (NV1 - 2); ++pr) exp_pair(pr);
          }
        });
        pfr[0] = __builtin_bit_cast(Frag, (u32x4){pw[0], pw[1], pw[2], pw[3]});
        mfma_trn_il<T, D>(vcur, vta, pfr, acc, [&](int i) {
#pragma unroll
          for (int pr = 4; pr < 16; ++pr) {
            const int f = pr >> 2, q4 = pr & 3;
            if (i == (f - 1) * NDT + (q4 * NDT) / 4) {
              exp_pair(pr);
              if (q4 == 3)
                pfr[f] = __builtin_bit_cast(Frag, (u32x4){pw[4 * f], pw[4 * f + 1], pw[4 * f + 2], pw[4 * f + 3]});
            }
          }
#pragma unroll
          for (int e = 0; e < VPS2; ++e) {
            const int v = i * VPS2 + e;
            mx = fmaxf(mx, s_nxt[v >> 4][v & 15]);
          }
          asm volatile("" : "+v"(mx));
        });
        l_run += rs;
        mx_carry = mx;
        if (masked) mx_carry = block_max(s_nxt, (j + 1) * kBN);
      } else {
#pragma unroll
        for (int i = 0; i < 2 * PT; ++i) load_part(i);
        __builtin_amdgcn_sched_barrier(0);
        update_max(wave_xor32_max(mx_carry) * c2);
        mfma_nat<T, D>(kcur, l32, hh, qf, s_nxt[0], s_nxt[1]);
        float rs = 0.f;
#pragma unroll
        for (int v = 0; v < 32; ++v) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s_cur[v >> 4][v & 15], c2, -m_run));
          s_cur[v >> 4][v & 15] = x;
          rs += x;
        }
        l_run += rs;
        pack_frags<T>(s_cur[0], s_cur[1], pfr);
        mfma_trn<T, D>(vcur, lane, vta, pfr, acc);
        mx_carry = block_max(s_nxt, (j + 1) * kBN);
      }
      s_cur[0] = s_nxt[0];
      s_cur[1] = s_nxt[1];
    }
#pragma unroll
    for (int u = 0; u < PT; ++u) row_v[u] = row_k[u];
    dma_wait();
    __syncthreads();
  }
  if (!active) return;

  update_max(wave_xor32_max(mx_carry) * c2);
  {
    Frag pfr[PF];
    float rs = 0.f;
#pragma unroll
    for (int v = 0; v < 32; ++v) {
      const float x = __builtin_amdgcn_exp2f(fmaf(s_cur[v >> 4][v & 15], c2, -m_run));
      s_cur[v >> 4][v & 15] = x;
      rs += x;
    }
    l_run += rs;
    pack_frags<T>(s_cur[0], s_cur[1], pfr);
    mfma_trn<T, D>(vbuf0 + ((nblk - 1) & 1) * G::BYTES, lane, vta, pfr, acc);
  }
  const float l_tot = wave_xor32_sum(l_run);
  if (r < n_rows) {
    const int64_t at = (int64_t)piece * p.B * p.Hq + (int64_t)b * p.Hq + h;
    store_acc_row<float, D>(p.part_o + at * D, acc, 1.f, hh);
    if (hh == 0) *reinterpret_cast<f32x2*>(p.part_ml + 2 * at) = (f32x2){m_run, l_tot};
  }
}

// The merge: a workgroup per (batch, kv head, 16 of its heads), D / 4 lanes a
// row, 16 bytes each; where the rows leave lanes over, groups of lanes share the
// chunks and join through LDS. Bound by the partials' latency: 8 are in flight
// per lane.
template <typename T, int D>
__global__ __launch_bounds__(256) void pf_prefix_merge_kernel(PrefixParams p) {
  constexpr int LPR = D / 4, NB = 8;
  const int g = p.g, n16 = (g + 15) >> 4, J = p.Hkv * n16;
  const int b = blockIdx.x / J, j = blockIdx.x - b * J;
  const int kvh = j / n16, hc = j - kvh * n16;
  const int nq = min(16, g - 16 * hc);
  const int tid = threadIdx.x;
  // the live chunks: of the prefix, then of the sequence
  const int npre = (prefix_len(p) + p.chunk - 1) / p.chunk;
  const int total = npre + (p.n_own > 0 ? (own_len(p, b) + p.own_chunk - 1) / p.own_chunk : 0);

  __shared__ f32x4 so[256];
  __shared__ f32x2 sm[256];
  const int per = nq * LPR;
  const int ngrp = per >= 256 ? 1 : 256 / per;
  const int grp = per >= 256 ? 0 : tid / per;
  for (int i0 = 0; i0 < per; i0 += 256) {  // one round where per <= 256
    const int i = per >= 256 ? i0 + tid : tid - grp * per;
    const bool on = i < per && grp < ngrp;
    const int qi = on ? i / LPR : 0, d0 = on ? 4 * (i % LPR) : 0;
    const int64_t bh = (int64_t)b * p.Hq + kvh * g + 16 * hc + qi;
    float M = kNegInf, l = 0.f;
    f32x4 o = (f32x4)(0.f);
    for (int c0 = grp; on && c0 < total; c0 += NB * ngrp) {
      f32x2 ml[NB];
      f32x4 v[NB];
      float Mn = M;
#pragma unroll
      for (int c = 0; c < NB; ++c) {
        const int s = c0 + c * ngrp;
        ml[c] = (f32x2){kNegInf, 0.f};
        v[c] = (f32x4)(0.f);
        if (s < total) {
          const int64_t row = (int64_t)(s < npre ? s : p.n_split + s - npre) * p.B * p.Hq + bh;
          ml[c] = *reinterpret_cast<const f32x2*>(p.part_ml + row * 2);
          v[c] = *reinterpret_cast<const f32x4*>(p.part_o + row * D + d0);
        }
        Mn = fmaxf(Mn, ml[c][0]);
      }
      const float Mu = (Mn == kNegInf) ? 0.f : Mn;
      const float back = exp2f(M - Mu);
      o *= back;
      l *= back;
#pragma unroll
      for (int c = 0; c < NB; ++c) {
        const float wt = exp2f(ml[c][0] - Mu);
        l += ml[c][1] * wt;
        o += v[c] * wt;
      }
      M = Mn;
    }
    if (ngrp > 1) {
      so[tid] = o;
      sm[tid] = (f32x2){M, l};
      __syncthreads();
      if (grp != 0) return;
      for (int k = 1; k < ngrp; ++k) M = fmaxf(M, sm[tid + k * per][0]);
      const float Mu = (M == kNegInf) ? 0.f : M;
      const float mine = exp2f(sm[tid][0] - Mu);
      o *= mine;
      l *= mine;
      for (int k = 1; k < ngrp; ++k) {
        const f32x2 x = sm[tid + k * per];
        const float wt = exp2f(x[0] - Mu);
        l += x[1] * wt;
        o += so[tid + k * per] * wt;
      }
    }
    if (on && d0 < p.dr) {
      const float inv = (l == 0.f) ? 0.f : 1.f / l;  // no key, or none that weighs: o = 0
      typedef T v4 __attribute__((ext_vector_type(4)));
      v4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = Elem<T>::from_f32(o[e] * inv);
      *reinterpret_cast<v4*>(static_cast<T*>(p.o) + bh * p.dr + d0) = y;
    }
  }
}

template <typename T, int D>
hipError_t launch_typed(const PrefixParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.n_pre + p.n_own * p.B * p.Hkv * p.n_hc));
  if (grid.x > 0) {
    if (p.dma) hipLaunchKernelGGL((pf_prefix_kernel<T, D, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((pf_prefix_kernel<T, D, false>), grid, dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((pf_prefix_merge_kernel<T, D>), dim3((unsigned)(p.B * p.Hkv * ((p.g + 15) / 16))), dim3(256), 0,
                     st, p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_dim(const PrefixParams& p, int D, hipStream_t st) {
  if (D == 64) return launch_typed<T, 64>(p, st);
  if (D == 128) return launch_typed<T, 128>(p, st);
  if constexpr (sizeof(T) == 2)
    if (D == 256) return launch_typed<T, 256>(p, st);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_prefix(const PrefixParams& p, int dtype, int D, hipStream_t stream) {
  switch (dtype) {
    case kF32: return launch_dim<float>(p, D, stream);
    case kBF16: return launch_dim<bf16_t>(p, D, stream);
    case kF16: return launch_dim<f16_t>(p, D, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pf
