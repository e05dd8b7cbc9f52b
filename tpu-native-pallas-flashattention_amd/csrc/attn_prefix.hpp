// Single-query attention of a batch that shares a prefix (gfx950): every
// sequence attends the prefix's pages and then its own.
//
//   o_b = softmax(scale q_b [K_prefix; K_b]^T) [V_prefix; V_b]
//
// A paged decode reads the prefix once per sequence. Here the B g query rows
// of a KV head (all sequences, g heads each) are one matrix against it. Two
// launches:
//  * pf_prefix_kernel. Its first workgroups take a prefix item each: 128 rows
//    of a KV head against one chunk of the prefix's keys. The others share the
//    sequences' own keys: the streaming decode's work list (decode_stream.hpp),
//    a contiguous run of it each, whatever the lengths. Prefix items are bound
//    by the matrix cores where there are many sequences, own keys by memory;
//    both kinds run beside each other. Each leaves (max, sum, acc) of its rows
//    in float32 for every chunk or piece.
//  * pf_prefix_merge_kernel: o = sum_i acc_i 2^(m_i - M) / sum_i l_i 2^(m_i - M)
//    over a row's chunks and pieces.
// No counterpart in the reference, whose paged call gives the prefix's pages
// to every sequence's table (paged.py:102-192).
//
// A prefix item runs the prefill forward's arithmetic (attn_fwd.hip) over pages:
// 64-key blocks in LDS, S^T = K Q^T of block t + 1 beside the exponentials of
// block t, O^T += V^T P^T of block t beside the maximum of block t + 1. Its keys
// come from memory, not from an L2 that many workgroups share, and the own keys
// beside it keep memory busy, so the loads run further ahead than there, in as
// many tiles (two of K, two of V): a second barrier, in the middle of a block,
// frees K_{t+1}'s tile for K_{t+3} while P.V of block t runs, and a wait is for the
// tile needed next alone. The tiles come by direct global -> LDS loads of whole
// rows (1 KB each; rows past the length and columns past the stored head dim lie
// outside the load's buffer range and arrive as zeros), one page lookup per wave
// and tile, two where 16 rows may straddle pages (50-row pages, 64 sequences of up
// to 2048 keys over 4000: 75 us, staged through registers 241). Small odd pages,
// such pools past 4 GiB and unaligned ones are staged through registers.
// Measured (bfloat16, head_dim 128, 32 heads over 8, 128 sequences, 32768 prefix
// keys): the prefix alone 94 us with an item per CU, 90 (764 TFLOP/s) with two. One
// wave a SIMD leaves the pipeline bound by its instructions and their latencies;
// what helped was one lookup and descriptor per tile and wave, tile addresses that
// are constants of each block's copy, nothing of the own keys' code in the loop (177
// us for prefix and own keys -> 144), and page lookups a block ahead (142 -> 136).
// With the own keys (4.3 MB a sequence, 96 us alone, 5.6 TB/s) 136 us: reads beside
// products that share the SIMDs. 32 sequences over 6000 keys: 31 us.
//
// Own keys with at most 16 heads a KV head: the workgroup's waves each stream a
// run of their own (key_stream). More heads, small odd pages and unaligned
// operands: the workgroup runs the prefix items' pipeline over its run, across the
// sequences: the block after a sequence's last one is the next sequence's first.
// float32 with at most 128 rows a KV head streams the prefix like own keys, 16 rows
// a wave (plan_prefix in capi.hip has the figures).
#pragma once

#include "decode_stream.hpp"
#include "pf_common.hpp"
#include "pf_kernels.hpp"
#include "pf_tiles.hpp"

namespace pf {

namespace prefix {

constexpr int kBN = 64;      // keys per block
constexpr int kRows = kPrefixRows;

constexpr uint32_t kPastRange = 0x7ffffff0u;  // an offset past any load's buffer range
constexpr uint32_t kPastPool = 0xfffffff0u;   // ... past any pool below 4 GiB
constexpr int kPG = 2;  // the work list's lengths are those of a paged call
using stream::Cursor;
typedef int i32x2 __attribute__((ext_vector_type(2)));

__device__ inline int prefix_len(const PrefixParams& p) {
  return p.len_ptr != nullptr ? min(max(stream::sload_i32(p.len_ptr, 0), 0), p.len) : p.len;
}

// Slot of an own piece of sequence seq that workgroup w leaves; whole: all of the
// sequence. Few sequences: w + seq names every piece once (stream::piece_slot).
// Many: a workgroup leaves at most a piece that opens its run and one that closes
// it, and whole sequences have slots of their own.
__device__ inline int64_t own_slot(const DecodeParams& p, int J, int w, int64_t seq, bool whole, bool late) {
  if (whole && (int64_t)p.B * J > p.n_waves) return 2 * (int64_t)p.n_waves + seq;
  return stream::piece_slot(p, J, w, seq, late);
}

// What the merge has to know of a sequence's own pieces, left by the workgroup or
// wave w whose piece opens it (c: that piece's last stage): w, whether the piece is
// not w's first, and how many pieces there are, w's and its successors'.
__device__ inline void own_note(const PrefixParams& p, const stream::Partition& part, int w, int64_t seq,
                                const Cursor& c, bool late) {
  int np = 1;
  if (c.st < c.nst - 1) np += part.wave_of(part.start(w + 1) + (c.nst - 2 - c.st)) - w;
  reinterpret_cast<i32x2*>(p.own_info)[seq] = (i32x2){2 * w + (late ? 1 : 0), np};
}

// Loads of 64-row tiles: the keys [64 st, ...) below L of the cursor's sequence.
// Wave w loads rows 16 w .. 16 w + 15. DMA > 0: whole rows by direct loads; 16:
// the wave's rows lie in one page (page_size % 16 == 0), so that a tile takes one
// lookup and one descriptor -- with a wave on each SIMD the scalar instructions of
// one per load cost as much as the exponentials; 2: they lie in at most two pages
// (page_size >= 16), and each lane picks its row's, by offsets in the whole pool
// (below 4 GiB); 1: each load's rows lie in one page. DMA = 0: every lane fetches
// its 16-byte chunks itself.
template <typename T, int D, int DMA>
struct PageTiles {
  using G = Tile<T, D>;
  static constexpr int PT = G::CPR / 4;          // loads per lane and tile
  static constexpr int RPL = 1024 / G::RB;       // rows per load
  static constexpr int GR = DMA == 16 ? 16 : DMA == 2 ? 15 : RPL;  // rows from lookup to lookup
  static constexpr int NG = DMA == 2 ? 2 : 16 / GR;                // lookups of a wave per tile
  uint32_t voff[PT];  // the lane's byte offset within the lookup's rows (DMA = 2: the wave's)
  uint32_t row0;      // the wave's first row; load u: + RPL u
  uint32_t slot0;     // the wave's LDS byte offset of load 0; load u: + 1024 u
  uint32_t rb;        // stored row bytes
  int lane, n_hc;
  const PrefixParams& p;
  const int32_t* table;  // of the prefix, or all sequences'
  int pages;             // per sequence

  __device__ inline PageTiles(const PrefixParams& p_, int tid, bool own)
      : rb(p_.dr * G::ES), lane(tid & 63), n_hc(own ? p_.n_hc : 1), p(p_),
        table(own ? p_.own.block_tables : p_.table), pages(own ? p_.own.pages_per_seq : p_.pages) {
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    row0 = 16 * w;
    slot0 = 1024 * PT * w;
#pragma unroll
    for (int u = 0; u < PT; ++u) {
      const int row = RPL * u + lane / G::CPR;
      const int chunk = (lane % G::CPR) ^ tile_swz<G::CPR>(16 * w + row);
      // columns past the stored row: past any range
      voff[u] = chunk * G::EPC < p.dr ? (uint32_t)(((DMA == 2 ? row : row % GR) * p.dr + chunk * G::EPC) * G::ES) : kPastRange;
    }
  }
  __device__ inline int kv_head(const Cursor& c) const { return n_hc == 1 ? c.j : c.j / n_hc; }
  // The pages of a block's lookups (wave-uniform: scalar loads of the table, which
  // do not disturb the count of the loads in flight), asked for a block before
  // rows() takes them. A lookup past the table's reach takes the last page and
  // reads nothing.
  struct Pages {
    int id[NG];
  };
  __device__ inline int key_of(const Cursor& c, int u) const {
    return kBN * c.st + row0 + GR * u;
  }
  __device__ inline int logical(int key) const { return min((int)fast_div(key, p.div_page), pages - 1); }
  __device__ inline Pages look(const Cursor& c) const {
    Pages x;
#pragma unroll
    for (int u = 0; u < NG; ++u) x.id[u] = stream::sload_i32(table, (int64_t)c.b * pages + logical(key_of(c, u)));
    return x;
  }
  // The byte offsets in the pool where they start, and the valid bytes behind them.
  // (DMA = 2: those of the wave's first row as if it lay in either page, modulo
  // 2^32, and the valid rows and those in the first page.)
  struct Rows {
    uint64_t at[NG];
    uint32_t bytes[NG];
  };
  __device__ inline Rows rows(const Cursor& c, const Pages& page) const {
    Rows x;
    const int kvh = kv_head(c);
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int key = key_of(c, u), id = min(max(page.id[u], 0), p.num_pages - 1);
      if constexpr (DMA == 2) {
        const int key0 = key_of(c, 0), first = logical(key) * p.page_size;
        x.at[u] = (((uint32_t)id * p.Hkv + kvh) * p.page_size + (uint32_t)(key0 - first)) * rb;
        x.bytes[u] = u == 0 ? min(max(c.L - key0, 0), 16) : logical(key0) * p.page_size + p.page_size - key0;
        continue;
      }
      x.at[u] = (uint64_t)(((uint32_t)id * p.Hkv + kvh) * p.page_size + (key - logical(key) * p.page_size)) * rb;
      x.bytes[u] = min(max(c.L - key, 0), GR) * rb;
    }
    return x;
  }
  // The descriptor of the wave's rows (DMA = 16; 2: of the pool), for all its loads.
  __device__ inline i32x4 rows_desc(const void* pool, const Rows& x) const {
    if constexpr (DMA == 2)
      return dma_pin(make_desc(pool, (uint32_t)p.num_pages * p.Hkv * p.page_size * rb));
    return dma_pin(make_desc(static_cast<const char*>(pool) + x.at[0], x.bytes[0]));
  }
  __device__ inline void load(const i32x4& pinned, const Rows& x, int u, char* tile) const {
    uint32_t at = voff[u];
    if constexpr (DMA == 2) {
      const uint32_t row = RPL * u + lane / G::CPR;
      at += row < x.bytes[1] ? (uint32_t)x.at[0] : (uint32_t)x.at[1];
      if (row >= x.bytes[0] || voff[u] == kPastRange) at = kPastPool;
    }
    dma16_pinned<true>(pinned, at, __builtin_amdgcn_readfirstlane(lds_u32(tile) + slot0 + 1024 * u));
  }
  __device__ inline void load(const void* pool, const Rows& x, int u, char* tile) const {
    const i32x4 d = make_desc(static_cast<const char*>(pool) + x.at[u], x.bytes[u]);
    dma16<true>(d, voff[u], __builtin_amdgcn_readfirstlane(lds_u32(tile) + slot0 + 1024 * u));
  }
  // Without DMA: a block through registers.
  __device__ inline void copy(const void* pool, const Cursor& c, char* tile) const {
    u32x4 x[PT];
#pragma unroll
    for (int u = 0; u < PT; ++u) {
      const int s = (slot0 + 1024 * u) / 16 + lane, row = s / G::CPR;
      const int chunk = (s % G::CPR) ^ tile_swz<G::CPR>(row), key = kBN * c.st + row;
      x[u] = (u32x4){0u, 0u, 0u, 0u};
      if (key < c.L && chunk * G::EPC < p.dr) {
        const int lp = fast_div(key, p.div_page);
        const int page = min(max(table[(int64_t)c.b * pages + lp], 0), p.num_pages - 1);
        const int64_t at = ((int64_t)page * p.Hkv + kv_head(c)) * p.page_size + (key - lp * p.page_size);
        x[u] = ldg16(static_cast<const T*>(pool) + at * p.dr + chunk * G::EPC);
      }
    }
#pragma unroll
    for (int u = 0; u < PT; ++u) sts16(tile + slot0 + 1024 * u + 16 * lane, x[u]);
  }
};

// ---------------------------------------------------------------------------
// Own keys, at most 16 query heads per KV head: wave w of own.n_waves streams its
// run of the work list in stages of 16 keys through a ring of two stages in LDS,
// with no barrier: 16x16 MFMAs, S^T (16 keys x heads) and O^T += V^T P^T, as the
// streaming decode. A stage's K is free once its scores are there, its V once
// P.V is, and each is refilled right then with the stage two on: two stages are
// in flight nearly always, 64 KB of a workgroup's four waves at head_dim 128.
// (Half of that, refilled stage by stage, or the prefix pipeline over 64-key
// blocks, is what leaves a CU that also computes a prefix item short of memory
// traffic.) A sequence's query rows come the same way, with its first stage, or,
// where those of a one-stage sequence still wait to be taken, right after them.
// PG: rows of one page lookup (page_size % PG == 0); kSplit: a stage lies in at
// most two pages and each lane picks its row's, as PageTiles with DMA = 2.
// ---------------------------------------------------------------------------
constexpr int kOwnKeys = 16;   // keys per stage
constexpr int kOwnHeads = 16;  // query rows per sequence, at most
constexpr int kSplit = 2;

template <typename T, int D>
struct OwnGeo {
  static constexpr int RB = D * (int)sizeof(T);  // row bytes: 128, 256 or 512
  static constexpr int CPR = RB / 16;            // chunks per row
  static constexpr int TILE = kOwnKeys * RB;     // a stage of K (or V)
  static constexpr int NL = TILE / 1024;         // loads per tile
  static constexpr int RPL = 1024 / RB;          // rows per load
  static constexpr int QB = kOwnHeads * RB;      // query rows
  static constexpr int WAVE = 4 * TILE + QB;     // K, V: two stages each; Q: one sequence
  static_assert(RB == 128 || RB == 256 || RB == 512, "row sizes");
  // Chunk permutation of row r (XOR of the low bits of the chunk index): the 16
  // rows of a K read hit 16 bank groups (128-byte rows: row bit 0 already parts
  // two rows of a bank window), and so do the 4 rows x 2 chunks of a V read.
  __host__ __device__ static constexpr int swz(int r) {
    if (RB == 128) return (((r >> 1) & 1) << 1) | ((r >> 3) & 1) | (((r >> 2) & 1) << 2);
    return ((r >> 2) & 1) | ((r & 3) << 1) | (((r >> 3) & 1) << 3);
  }
  static constexpr int QMASK = (CPR < 16 ? CPR : 16) - 1;  // query row permutation
};

// The wave's LDS reads so far have their data (what they read may be overwritten).
__device__ inline void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// PRE (float32, few rows): w's item of the prefix instead, 16 of a KV head's rows
// against one chunk of its keys.
template <typename T, int D, int PG, bool PRE>
__device__ __forceinline__ void key_stream(const PrefixParams& p, char* ring, int w) {
  using MF = stream::Mfma16<T>;
  using G = OwnGeo<T, D>;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int SK = kOwnKeys, RB = G::RB, NL = G::NL, NSTEP = G::CPR / 4, NACC = D / 16;
  constexpr bool SPLIT = PG == kSplit;
  constexpr int kGroups = SPLIT ? 2 : SK / PG, kPer = SPLIT ? NL : NL / kGroups;
  static_assert(SPLIT || (PG % G::RPL == 0 && SK % PG == 0), "a page group is whole loads of one stage");
  const DecodeParams& own = p.own;
  const int lane = threadIdx.x & 63, i16 = lane & 15, h = lane >> 4;
  const int J = p.Hkv, ps = p.page_size;
  const int32_t* const table = PRE ? p.table : own.block_tables;
  const int pages = PRE ? p.pages : own.pages_per_seq;

  Cursor cc;
  [[maybe_unused]] stream::Partition part((int64_t)0, (int64_t)0);
  int64_t n;
  int r0 = 0, piece = 0;  // PRE: the item's first row, and its chunk
  if constexpr (PRE) {
    // The waves of a workgroup: row groups, then chunks of one KV head, which is
    // the workgroups' innermost index.
    const int wg = w >> 2, kvh = wg % J, y = 4 * (wg / J) + (w & 3);
    piece = y / p.n_tiles;
    r0 = kOwnHeads * (y - piece * p.n_tiles);
    // Waves past the last item have nothing (and a key0 past 32 bits).
    const bool on = piece < p.n_split;
    const int key0 = on ? piece * p.chunk : 0, L = on ? min(prefix_len(p), key0 + p.chunk) : 0;
    n = (L - key0 + SK - 1) / SK;
    cc = Cursor{0, kvh, key0 / SK, key0 / SK + (int)n, L};
  } else {
    if (w >= own.n_waves) return;
    n = stream::wave_plan<kPG, SK>(own, J, own.n_waves, w, &cc, &part);
  }
  if (n <= 0) return;
  const int g = PRE ? min(p.rows - r0, kOwnHeads) : p.g;  // query rows
  auto next = [&](Cursor& c) {
    if constexpr (PRE) ++c.st;
    else stream::cursor_next<kPG, SK>(c, own, J);
  };
  // PRE: the (batch, head) of the item's row.
  auto head_of = [&](int row) {
    const int b = (r0 + row) / p.g;
    return b * p.Hq + cc.j * p.g + (r0 + row - b * p.g);
  };

  char* const kbuf = ring;                 // stages k & 1
  char* const vbuf = ring + 2 * G::TILE;
  char* const qbuf = ring + 4 * G::TILE;

  // The chunk that this lane fetches for load i: its byte offset within the page group.
  // (Columns past the stored row: past any range.)
  const uint32_t rb = p.dr * sizeof(T);
  uint32_t loff[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int row = G::RPL * i + lane / G::CPR;
    const uint32_t at = 16 * ((lane % G::CPR) ^ G::swz(row));
    loff[i] = at < rb ? (SPLIT ? row : row % PG) * rb + at : kPastRange;
  }
  // A stage's page groups: pool row and valid rows of each. Groups past the
  // length load nothing and look nothing up (-1 padding). SPLIT: the pool row of
  // the stage's first key as if it lay in the page of the first, or the last, valid
  // key (modulo 2^32); its valid keys and those in the first page.
  struct Stage {
    uint32_t row[kGroups];
    int valid[kGroups];
  };
  auto look = [&](const Cursor& c) {
    Stage s;
    if constexpr (SPLIT) {
      const int key0 = c.st * SK, n = min(c.L - key0, SK);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int lp = fast_div(i == 0 ? key0 : key0 + n - 1, p.div_page);
        int page = stream::sload_i32(table, (int64_t)c.b * pages + lp);
        page = min(max(page, 0), p.num_pages - 1);
        s.row[i] = ((uint32_t)page * p.Hkv + c.j) * ps + (uint32_t)(key0 - lp * ps);
        s.valid[i] = i == 0 ? n : (int)fast_div(key0, p.div_page) * ps + ps - key0;
      }
      return s;
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int key = c.st * SK + i * PG;
      s.valid[i] = min(max(c.L - key, 0), PG);
      const int lp = s.valid[i] > 0 ? (int)fast_div(key, p.div_page) : 0;
      int page = s.valid[i] > 0 ? stream::sload_i32(table, (int64_t)c.b * pages + lp) : 0;
      page = min(max(page, 0), p.num_pages - 1);
      s.row[i] = ((uint32_t)page * p.Hkv + c.j) * ps + (s.valid[i] > 0 ? key - lp * ps : 0);
    }
    return s;
  };
  auto load = [&](const void* pool, const Stage& s, char* tile) {
    const uint32_t at = lds_u32(tile);
    if constexpr (SPLIT) {
      const i32x4 d = dma_pin(make_desc(pool, (uint32_t)p.num_pages * p.Hkv * ps * rb));
      const uint32_t r0 = s.row[0] * rb, r1 = s.row[1] * rb;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int row = G::RPL * i + lane / G::CPR;
        const uint32_t off = loff[i] + (row < s.valid[1] ? r0 : r1);
        dma16_pinned<true>(d, row < s.valid[0] && loff[i] != kPastRange ? off : kPastPool, at + 1024 * i);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const i32x4 d = make_desc(static_cast<const char*>(pool) + (uint64_t)s.row[i] * rb, s.valid[i] * rb);
#pragma unroll
      for (int e = 0; e < kPer; ++e) dma16<true>(d, loff[i * kPer + e], at + 1024 * (i * kPer + e));
    }
  };
  // q_wait: the queries in qbuf are still to be taken; qb, qj: the sequence whose
  // queries come after those (qb < 0: none).
  bool q_wait = false;
  int qb = -1, qj = 0;
  auto load_q = [&](int b, int j) {
    if (q_wait) {
      qb = b;
      qj = j;
      return;
    }
    q_wait = true;
    const i32x4 d = PRE ? make_desc(p.q, (uint32_t)own.B * p.Hq * rb)
                        : make_desc(static_cast<const T*>(p.q) + ((int64_t)b * p.Hq + (int64_t)j * g) * p.dr, g * rb);
#pragma unroll
    for (int i = 0; i < G::QB / 1024; ++i) {
      const int row = G::RPL * i + lane / G::CPR;
      const uint32_t at = 16 * ((lane % G::CPR) ^ (row & G::QMASK));
      const bool on = at < rb && (!PRE || row < g);
      if (G::RPL * i < g) dma16(d, on ? (PRE ? head_of(row) : row) * rb + at : kPastRange, lds_u32(qbuf) + 1024 * i);
    }
  };

  // Prologue: stages 0 and 1. pc: the stage that is loaded next.
  Cursor pc = cc;
  load_q(cc.b, cc.j);
  Stage st = look(cc);
  load(p.k, st, kbuf);
  load(p.v, st, vbuf);
  next(pc);
  if (n > 1) {
    st = look(pc);
    if (!PRE && pc.st == 0) load_q(pc.b, pc.j);
    load(p.k, st, kbuf + G::TILE);
    load(p.v, st, vbuf + G::TILE);
    next(pc);
  }

  // LDS read offsets. K (A operand of S^T): row i16, chunk 4s + h; past 16 chunks
  // 256 bytes on. V: 16-bit, transposing reads of rows 4h + i16/4, columns 16dt +
  // 4(i16%4) .. + 3; float32, row 4h + e, chunk i16.
  constexpr int NKO = NSTEP < 4 ? NSTEP : 4, NVO = F32 ? 4 : (NACC < 8 ? NACC : 8);
  uint32_t koff[NKO], voff[NVO];
#pragma unroll
  for (int s = 0; s < NKO; ++s) koff[s] = (uint32_t)(i16 * RB + 16 * ((4 * s + h) ^ G::swz(i16)));
#pragma unroll
  for (int e = 0; e < NVO; ++e) {
    if constexpr (F32) {
      voff[e] = (uint32_t)((4 * h + e) * RB + 16 * (i16 ^ G::swz(4 * h + e)));
    } else {
      const int row = 4 * h + (i16 >> 2), chunk = 2 * e + ((i16 >> 1) & 1);
      voff[e] = (uint32_t)(row * RB + 16 * (chunk ^ G::swz(row)) + 8 * (i16 & 1));
    }
  }

  u32x4 qf[NSTEP];
  // O^T: 16-bit tile dt, register r = column 16dt + 4h + r; float32 tile 4 blk + e,
  // register r = column 64 blk + 16h + 4r + e. Column i16: head i16.
  f32x4 acc[NACC];
  float m_run = -__FLT_MAX__, l_run = 0.f;  // as the prefix items
  int piece_st0 = 0;
  bool first_piece = true;

  for (int64_t k = 0; k < n; ++k) {
    // Loads complete in order: all but the next stage's (queries with its first
    // one included) are there.
    if (k + 1 < n) wait_vm<2 * NL>();
    else wait_vm<0>();
    char* const sK = kbuf + (k & 1) * G::TILE;
    char* const sV = vbuf + (k & 1) * G::TILE;
    if (k == 0 || (!PRE && cc.st == 0)) {
#pragma unroll
      for (int s = 0; s < NSTEP; ++s)
        qf[s] = i16 < g ? lds16(qbuf + i16 * RB + 16 * ((4 * s + h) ^ (i16 & G::QMASK))) : (u32x4){0u, 0u, 0u, 0u};
      q_wait = false;
      if (qb >= 0) {
        wait_lds();
        load_q(qb, qj);
        qb = -1;
      }
#pragma unroll
      for (int a = 0; a < NACC; ++a) acc[a] = (f32x4)(0.f);
      m_run = -__FLT_MAX__;
      l_run = 0.f;
      piece_st0 = cc.st;
    }
    f32x4 s = (f32x4)(0.f);  // keys 4h + r, head i16
#pragma unroll
    for (int e = 0; e < NSTEP; ++e) s = MF::run(lds16(sK + koff[e % NKO] + 256 * (e / NKO)), qf[e], s);

    const bool more = k + 2 < n;
    if (more) {
      st = look(pc);
      wait_lds();  // K and Q are read
      if (!PRE && pc.st == 0) load_q(pc.b, pc.j);
      load(p.k, st, sK);
    }

    float x[4], mx = kNegInf;
    const int rel = cc.L - cc.st * SK - 4 * h;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x[t] = t < rel ? s[t] * p.scale_log2 : kNegInf;
      mx = fmaxf(mx, x[t]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = wave_xor32_max(mx);
    const float m_cand = fmaxf(m_run, mx);
    if (__any(m_cand > m_run + 8.f)) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_cand);
#pragma unroll
      for (int a = 0; a < NACC; ++a) acc[a] *= alpha;
      l_run *= alpha;
      m_run = m_cand;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x[t] = __builtin_amdgcn_exp2f(x[t] - m_run);
      l_run += x[t];
    }
    if constexpr (F32) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int blk = 0; blk < D / 64; ++blk) {
          const f32x4 v = __builtin_bit_cast(f32x4, lds16(sV + voff[t] + 256 * blk));
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[4 * blk + e] = MF::step(v[e], x[t], acc[4 * blk + e]);
        }
    } else {
      const u32x2 pf = {pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};  // half a step of each weight
#pragma unroll
      for (int dt = 0; dt < NACC; ++dt) {
        const stream::i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) stream::i16x4*)(sV + voff[dt % NVO] + 256 * (dt / NVO)));
        acc[dt] = MF::run16(__builtin_bit_cast(u32x2, v), pf, acc[dt]);
      }
    }
    if (more) {
      wait_lds();  // V is read
      load(p.v, st, sV);
      next(pc);
    }

    if ((!PRE && cc.st == cc.nst - 1) || k == n - 1) {
      float l_tot = l_run + __shfl_xor(l_run, 16);
      l_tot = wave_xor32_sum(l_tot);
      if (i16 < g) {
        int64_t at;
        if constexpr (PRE) {
          at = (int64_t)piece * own.B * p.Hq + head_of(i16);
        } else {
          const bool whole = piece_st0 == 0 && cc.st == cc.nst - 1;
          const int64_t seq = (int64_t)cc.b * J + cc.j;
          if (piece_st0 == 0 && lane == 0) own_note(p, part, w, seq, cc, !first_piece);
          at = own_slot(own, J, w, seq, whole, !first_piece) * g + i16;
        }
        float* po = (PRE ? p.part_o : own.part_o) + at * D;
#pragma unroll
        for (int q = 0; q < NACC; ++q) {
          if constexpr (F32) {
            const int blk = q >> 2, r = q & 3;
            *reinterpret_cast<f32x4*>(po + 64 * blk + 16 * h + 4 * r) =
                (f32x4){acc[4 * blk][r], acc[4 * blk + 1][r], acc[4 * blk + 2][r], acc[4 * blk + 3][r]};
          } else {
            *reinterpret_cast<f32x4*>(po + 16 * q + 4 * h) = acc[q];
          }
        }
        if (h == 0) *reinterpret_cast<f32x2*>((PRE ? p.part_ml : own.part_ml) + 2 * at) = (f32x2){m_run, l_tot};
      }
      first_piece = false;
    }
    next(cc);
  }
}

// The block pipeline of one workgroup: a prefix item, or (OWN) its run of the
// sequences' own keys. item: the workgroup's place among those of its kind.
template <typename T, int D, int DMA, bool OWN>
__device__ __forceinline__ void run_blocks(const PrefixParams& p, char* smem, int item) {
  using MF = Mfma32<T>;
  using Frag = typename MF::Frag;
  using G = Tile<T, D>;
  using PTiles = PageTiles<T, D, DMA>;
  constexpr int HALF = D / 2, EPC = G::EPC, FPC = frags_per_chunk<T>();
  constexpr int QF = HALF / MF::kK, NDT = D / 32, PF = 32 / MF::kK, PT = PTiles::PT;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hh = lane >> 5, l32 = lane & 31;
  const int J = p.Hkv * p.n_hc;

  // The workgroup's n blocks and the first one's cursor.
  Cursor cp;
  int n, r0 = 0, piece = 0;
  [[maybe_unused]] stream::Partition part((int64_t)0, (int64_t)0);
  if constexpr (!OWN) {
    // (chunk, kv head, row tile): the row tiles of one chunk side by side on one
    // XCD, whose L2 then serves the chunk to all of them.
    const int it = xcd_remap(item, p.n_pre, p.n_tiles);
    r0 = kRows * (it % p.n_tiles);
    piece = it / p.n_tiles / p.Hkv;
    const int key0 = piece * p.chunk, L = min(prefix_len(p), key0 + p.chunk);
    n = (L - key0 + kBN - 1) / kBN;
    cp = Cursor{0, it / p.n_tiles % p.Hkv, key0 / kBN, key0 / kBN + n, L};
  } else {
    n = (int)stream::wave_plan<kPG, kBN>(p.own, J, p.own.n_waves, item, &cp, &part);
  }
  n = __builtin_amdgcn_readfirstlane(n);  // barriers are counted by it
  if (n <= 0) return;

  const PTiles tiles(p, tid, OWN);
  // The cursor of the block after c's (block t of the run); past the run, one whose
  // loads read nothing: every block issues the same loads, so that the waits can
  // count them.
  auto after = [&](Cursor c, int t) {
    if (t + 1 >= n) c.L = 0;
    else if constexpr (OWN) stream::cursor_next<kPG, kBN>(c, p.own, J);
    else ++c.st;
    return c;
  };

  // An own block seldom has rows for more than one wave: which one differs from
  // workgroup to workgroup, so that those on a CU load all of its SIMDs.
  const int w32 = 32 * (OWN ? (wv + item) & 3 : wv);
  // The lane's query row in the cursor's sequence: (batch, head) index, or -1.
  auto row_of = [&](const Cursor& c) -> int {
    if constexpr (!OWN) {
      const int r = r0 + w32 + l32;
      if (r >= p.rows) return -1;
      const int b = r / p.g;
      return b * p.Hq + c.j * p.g + (r - b * p.g);
    } else {
      const int kvh = tiles.kv_head(c), r = kRows * (c.j - kvh * p.n_hc) + w32 + l32;
      return r < p.g ? c.b * p.Hq + kvh * p.g + r : -1;
    }
  };

  // Cursors of blocks t (cp) .. t + 4 (cm), where the loads of blocks t + 1 .. t + 3
  // start, and the pages of block t + 4.
  char* const kbuf = smem;  // K tiles t & 1, then V tiles
  char* const vbuf = smem + 2 * G::BYTES;
  Cursor cs = after(cp, 0), ck = after(cs, 1), cl = after(ck, 2), cm = after(cl, 3);
  typename PTiles::Rows r1, r2, r3;
  typename PTiles::Pages next;
  auto whole = [&](const void* pool, [[maybe_unused]] const Cursor& c, const typename PTiles::Rows& x, char* tile) {
    if constexpr (DMA > 1) {
      const i32x4 d = tiles.rows_desc(pool, x);
#pragma unroll
      for (int u = 0; u < PT; ++u) tiles.load(d, x, u, tile);
    } else if constexpr (DMA > 0) {
#pragma unroll
      for (int u = 0; u < PT; ++u) tiles.load(pool, x, u, tile);
    } else {
      tiles.copy(pool, c, tile);
    }
  };
  {
    typename PTiles::Rows r;
    if constexpr (DMA > 0) {
      const auto p0 = tiles.look(cp), p1 = tiles.look(cs), p2 = tiles.look(ck), p3 = tiles.look(cl);
      next = tiles.look(cm);
      r = tiles.rows(cp, p0);
      r1 = tiles.rows(cs, p1);
      r2 = tiles.rows(ck, p2);
      r3 = tiles.rows(cl, p3);
    }
    whole(p.k, cp, r, kbuf);
    whole(p.k, cs, r1, kbuf + G::BYTES);
    whole(p.v, cp, r, vbuf);
  }
  // Block t, P = t & 1 (the tiles' addresses are constants of each copy): V_{t+1},
  // beside S_{t+1}, goes where V_{t-1} was, K_{t+3}, beside P.V, where K_{t+1} was.
  auto kcur = [&](auto par) { return kbuf + (1 - decltype(par)::value) * G::BYTES; };
  auto vcur = [&](auto par) { return vbuf + decltype(par)::value * G::BYTES; };
  auto vdst = [&](auto par) { return vbuf + (1 - decltype(par)::value) * G::BYTES; };
  i32x4 vd, kd;
  auto begin = [&](auto par) __attribute__((always_inline)) {
    if constexpr (DMA > 1) {
      vd = tiles.rows_desc(p.v, r1);
      kd = tiles.rows_desc(p.k, r3);
    }
    if constexpr (DMA == 0) tiles.copy(p.v, cs, vdst(par));
  };
  auto v_part = [&](int i, auto par) __attribute__((always_inline)) {
    if constexpr (DMA > 1) tiles.load(vd, r1, i, vdst(par));
    else if constexpr (DMA > 0) tiles.load(p.v, r1, i, vdst(par));
  };
  auto k_part = [&](int i, auto par) __attribute__((always_inline)) {
    if constexpr (DMA > 1) tiles.load(kd, r3, i, kcur(par));
    else if constexpr (DMA > 0) tiles.load(p.k, r3, i, kcur(par));
  };
  // The middle: V_t is there (after it K_{t+2} and V_{t+1} were asked for), and
  // every wave is done with K_{t+1}.
  auto middle = [&](auto par) __attribute__((always_inline)) {
    wait_vm<2 * PT>();
    __syncthreads();
    if constexpr (DMA == 0) tiles.copy(p.k, cl, kcur(par));
  };
  auto end = [&](int t) __attribute__((always_inline)) {
    cp = cs;
    cs = ck;
    ck = cl;
    cl = cm;
    cm = after(cm, t + 4);
    if constexpr (DMA > 0) {
      r1 = r2;
      r2 = r3;
      r3 = tiles.rows(cl, next);
      next = tiles.look(cm);
    }
    wait_vm<2 * PT>();  // K_{t+2}: V_{t+1} and K_{t+3} were asked for after it
    __syncthreads();
  };
  auto all_blocks = [&](auto&& block) __attribute__((always_inline)) {
    int t = 0;
    for (; t + 2 < n; t += 2) {
      block(t, std::integral_constant<int, 0>{});
      block(t + 1, std::integral_constant<int, 1>{});
    }
    if (t + 1 < n) block(t, std::integral_constant<int, 0>{});
  };

  // A wave without rows loads its share, and meets the others' barriers. (Of an
  // own sequence's slices only the last can be short.)
  const bool active = __builtin_amdgcn_readfirstlane(OWN ? w32 < p.own_rows : r0 + w32 < p.rows) != 0;
  if (!active) {
    dma_wait();
    __syncthreads();
    __syncthreads();
    whole(p.k, ck, r2, kbuf);
    all_blocks([&](int t, auto par) __attribute__((always_inline)) {
      begin(par);
#pragma unroll
      for (int i = 0; i < PT; ++i) v_part(i, par);
      middle(par);
#pragma unroll
      for (int i = 0; i < PT; ++i) k_part(i, par);
      end(t);
    });
    wait_vm<0>();
    __syncthreads();
    return;
  }

  u32x4 qc[HALF / EPC];  // Q: the lane's row, columns [hh HALF, + HALF)
  auto load_q = [&](const Cursor& c) __attribute__((always_inline)) {
    const int r = row_of(c);
    const T* qr = static_cast<const T*>(p.q) + (int64_t)r * p.dr + hh * HALF;
#pragma unroll
    for (int i = 0; i < HALF / EPC; ++i)
      qc[i] = r >= 0 && hh * HALF + i * EPC < p.dr ? ldg16(qr + i * EPC) : (u32x4){0u, 0u, 0u, 0u};
  };
  // A negative scale is applied as |scale| on -Q.
  auto sign_q = [&]() __attribute__((always_inline)) {
    if (p.scale_log2 < 0.f) {
      const uint32_t sign = G::ES == 4 ? 0x80000000u : 0x80008000u;
#pragma unroll
      for (int i = 0; i < HALF / EPC; ++i) qc[i] ^= (u32x4){sign, sign, sign, sign};
    }
  };
  auto frags = [&](Frag* qf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < HALF / EPC; ++i)
#pragma unroll
      for (int f = 0; f < FPC; ++f) qf[i * FPC + f] = chunk_frag<T>(qc[i], f);
  };
  load_q(cp);

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
  auto update_max = [&](float mx) __attribute__((always_inline)) {
    const float m_cand = fmaxf(m_run, mx);
    if (__any(m_cand > m_run + 8.f)) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_cand);
#pragma unroll
      for (int i = 0; i < NDT; ++i) acc[i] *= alpha;
      l_run *= alpha;
      m_run = m_cand;
    }
  };
  // The lane's maximum of a block's scores; keys at or past L become -inf.
  auto block_max = [&](f32x16* s, const Cursor& c) __attribute__((always_inline)) {
    const int rel = c.L - kBN * c.st - 32 * hh;
    float mx = kNegInf;
#pragma unroll
    for (int v = 0; v < 32; ++v) {
      const float x = v < rel ? s[v >> 4][v & 15] : kNegInf;
      s[v >> 4][v & 15] = x;
      mx = fmaxf(mx, x);
    }
    return mx;
  };
  // The end of a chunk or piece: its partials, and a fresh state.
  [[maybe_unused]] bool first_piece = true;
  [[maybe_unused]] int piece_st0 = cp.st;
  auto finish = [&](const Cursor& c) __attribute__((always_inline)) {
    const float l_tot = wave_xor32_sum(l_run);
    const int r = row_of(c);
    if (r >= 0) {
      float *po = p.part_o, *pm = p.part_ml;
      int64_t at = (int64_t)piece * p.own.B * p.Hq + r;
      if constexpr (OWN) {
        const int64_t seq = (int64_t)c.b * J + c.j;
        const bool whole_seq = piece_st0 == 0 && c.st == c.nst - 1;
        if (piece_st0 == 0 && w32 == 0 && lane == 0) own_note(p, part, item, seq, c, !first_piece);
        at = own_slot(p.own, J, item, seq, whole_seq, !first_piece) * p.own_rows + w32 + l32;
        po = p.own.part_o;
        pm = p.own.part_ml;
      }
      store_acc_row<float, D>(po + at * D, acc, 1.f, hh);
      if (hh == 0) *reinterpret_cast<f32x2*>(pm + 2 * at) = (f32x2){m_run, l_tot};
    }
    if constexpr (OWN) {
      first_piece = false;
      piece_st0 = 0;
      m_run = -__FLT_MAX__;
      l_run = 0.f;
#pragma unroll
      for (int i = 0; i < NDT; ++i) acc[i] = (f32x16)(0.f);
    }
  };

  dma_wait();
  __syncthreads();
  f32x16 s_cur[2] = {(f32x16)(0.f), (f32x16)(0.f)};
  // The lane's maximum of the latest block, not yet applied. A block that the
  // length cuts is masked when it is the run's last (before its exponentials), and
  // at a sequence's end (OWN).
  float mx_carry;
  {
    sign_q();
    Frag qf[QF];
    frags(qf);
    mfma_nat<T, D>(kbuf, l32, hh, qf, s_cur[0], s_cur[1]);
    mx_carry = block_max(s_cur, cp);
    if (OWN && n > 1 && cs.st == 0) {
      load_q(cs);
      sign_q();
    }
  }
  __syncthreads();  // K_0 is read before K_2 overwrites it
  whole(p.k, ck, r2, kbuf);

  all_blocks([&](int t, auto par) __attribute__((always_inline)) {
    const bool new_q = OWN && t + 2 < n && ck.st == 0;  // block t + 2 opens a sequence
    f32x16 s_nxt[2] = {(f32x16)(0.f), (f32x16)(0.f)};
    Frag qf[QF], pfr[PF];
    frags(qf);
    begin(par);
    if constexpr (sizeof(T) == 2) {
      // As in the forward: S_{t+1} beside the maximum and the first quarter of
      // S_t's exponentials, P.V beside the rest.
      constexpr int NV1 = G::CPR, NV2 = 4 * NDT, VPS2 = 32 / NV2;
      uint32_t pw[16];
      float rs = 0.f, mxr = kNegInf, mx = kNegInf;
      auto exp_pair = [&](int pr) __attribute__((always_inline)) {
        const int v = 2 * pr;
        const float x0 = __builtin_amdgcn_exp2f(fmaf(s_cur[v >> 4][v & 15], c2, -m_run));
        const float x1 = __builtin_amdgcn_exp2f(fmaf(s_cur[v >> 4][(v & 15) + 1], c2, -m_run));
        pw[pr] = pack2<T>(x0, x1);  // the matrix cores take P in T: half a step of each weight
        rs += x0 + x1;              // the sum is of the unrounded weights
        asm volatile("" : "+v"(rs));  // keeps the sum beside its MFMA
      };
      mfma_nat_il<T, D>(kcur(par), l32, hh, qf, s_nxt[0], s_nxt[1], [&](int i) {
        if (i < PT) v_part(i, par);
        if (i == 0) {
          mxr = wave_xor32_max(mx_carry) * c2;
        } else if (i == 1) {
          update_max(mxr);
        } else {
#pragma unroll
          for (int pr = ((i - 2) * 4) / (NV1 - 2); pr < ((i - 1) * 4) / (NV1 - 2); ++pr) exp_pair(pr);
        }
      });
      if (new_q) load_q(ck);  // Q is free now; there by the end of the block
      middle(par);
      pfr[0] = __builtin_bit_cast(Frag, (u32x4){pw[0], pw[1], pw[2], pw[3]});
      mfma_trn_il<T, D>(vcur(par), vta, pfr, acc, [&](int i) {
        if (i < PT) k_part(i, par);
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
    } else {
#pragma unroll
      for (int i = 0; i < PT; ++i) v_part(i, par);
      __builtin_amdgcn_sched_barrier(0);
      update_max(wave_xor32_max(mx_carry) * c2);
      mfma_nat<T, D>(kcur(par), l32, hh, qf, s_nxt[0], s_nxt[1]);
      if (new_q) load_q(ck);
      float rs = 0.f, mx = kNegInf;
#pragma unroll
      for (int v = 0; v < 32; ++v) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s_cur[v >> 4][v & 15], c2, -m_run));
        s_cur[v >> 4][v & 15] = x;
        rs += x;
      }
      l_run += rs;
      pack_frags<T>(s_cur[0], s_cur[1], pfr);
      middle(par);
#pragma unroll
      for (int i = 0; i < PT; ++i) k_part(i, par);
      mfma_trn<T, D>(vcur(par), lane, vta, pfr, acc);
#pragma unroll
      for (int v = 0; v < 32; ++v) mx = fmaxf(mx, s_nxt[v >> 4][v & 15]);
      mx_carry = mx;
    }
    if constexpr (OWN) {
      if ((cs.st + 1) * kBN > cs.L) mx_carry = block_max(s_nxt, cs);
      if (cp.st == cp.nst - 1) finish(cp);
      if (new_q) sign_q();
    }
    s_cur[0] = s_nxt[0];
    s_cur[1] = s_nxt[1];
    end(t);
  });
  wait_vm<0>();
  __syncthreads();

  update_max(wave_xor32_max(block_max(s_cur, cp)) * c2);
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
    mfma_trn<T, D>(vbuf + ((n - 1) & 1) * G::BYTES, lane, vta, pfr, acc);
  }
  finish(cp);
}

// PG > 0: own keys by key_stream; 0: by the block pipeline.
// The own pipeline needs the registers of two workgroups per CU at most.
template <typename T, int D, int DMA, int PG>
__global__ __launch_bounds__(256, (PG == 0 && kFwdWgPerCu<T, D> > 2 ? 2 : kFwdWgPerCu<T, D>))
void pf_prefix_kernel(PrefixParams p) {
  using G = OwnGeo<T, D>;
  static_assert(4 * G::WAVE >= 4 * Tile<T, D>::BYTES, "the waves' rings hold the tiles");
  __shared__ __attribute__((aligned(1024))) char smem[PG > 0 ? 4 * G::WAVE : 4 * Tile<T, D>::BYTES];
  const int item = blockIdx.x - p.n_pre;
  if constexpr (PG > 0) {
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* const ring = smem + wv * G::WAVE;
    if (item >= 0) return key_stream<T, D, PG, false>(p, ring, 4 * item + wv);
    if constexpr (sizeof(T) == 4)
      if (p.few) return key_stream<T, D, PG, true>(p, ring, 4 * blockIdx.x + wv);
  }
  if (item < 0) {
    run_blocks<T, D, DMA, false>(p, smem, blockIdx.x);
  } else if constexpr (PG == 0) {
    run_blocks<T, D, DMA, true>(p, smem, item);
  }
}

// The merge: a workgroup per (batch, kv head, merge_heads of its heads), D / 4
// lanes a row, 16 bytes each; groups of lanes share the chunks and pieces and join
// through LDS. The kv head is the innermost index, as that of the prefix items: an
// XCD mostly reads what its own L2 still holds (31 chunks of 192 keys, 32 sequences,
// both launches: 29 -> 21 us). Bound by latency: the chunks' partials, 8 in flight
// per lane, are on their way while the note of the own pieces comes.
// merge_heads is such that the chunks are one round of loads, where it can be.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void pf_prefix_merge_kernel(PrefixParams p) {
  constexpr int LPR = D / 4, NB = kMergeLoads;
  const int g = p.g, nh = p.merge_heads, n_h = (g + nh - 1) / nh;
  const int part = blockIdx.x / p.Hkv, kvh = blockIdx.x - part * p.Hkv;
  const int b = part / n_h, h0 = nh * (part - b * n_h);  // heads [h0, + nq) of the group
  const int nq = min(nh, g - h0);
  const int tid = threadIdx.x;
  const int per = nq * LPR, ngrp = 256 / per;  // per <= 256
  const int grp = tid / per, i = tid - grp * per, qi = i / LPR, d0 = 4 * (i - LPR * qi);
  const bool on = grp < ngrp;

  float M = kNegInf, l = 0.f;
  f32x4 o = (f32x4)(0.f);
  f32x2 ml[NB];
  f32x4 v[NB];
  // Partials grp, grp + ngrp, ... of [s0, total): row(s) of po and pm.
  auto fetch = [&](int s0, int total, const float* po, const float* pm, auto&& row) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < NB; ++c) {
      const int s = s0 + grp + c * ngrp;
      ml[c] = (f32x2){kNegInf, 0.f};
      v[c] = (f32x4)(0.f);
      if (on && s < total) {
        const int64_t r = row(s);
        ml[c] = *reinterpret_cast<const f32x2*>(pm + r * 2);
        v[c] = *reinterpret_cast<const f32x4*>(po + r * D + d0);
      }
    }
  };
  auto join = [&]() __attribute__((always_inline)) {
    float Mn = M;
#pragma unroll
    for (int c = 0; c < NB; ++c) Mn = fmaxf(Mn, ml[c][0]);
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
  };

  const int npre = prefix_chunks(prefix_len(p), p.chunk);
  const int64_t bh = (int64_t)b * p.Hq + kvh * g + h0 + qi;
  auto chunk_row = [&](int s) { return (int64_t)s * p.own.B * p.Hq + bh; };
  fetch(0, npre, p.part_o, p.part_ml, chunk_row);

  // The sequence's pieces, if it has keys (else nothing was noted).
  const int J = p.Hkv * p.n_hc, slice = h0 / kRows;
  const int64_t seq = (int64_t)b * J + kvh * p.n_hc + slice;
  i32x2 note = (i32x2){0, 0};
  if (p.own.n_waves > 0) {
    note = reinterpret_cast<const i32x2*>(p.own_info)[seq];
    if (stream::seq_len<kPG>(p.own, b) <= 0) note = (i32x2){0, 0};
  }
  const int wa = note[0] >> 1, np = note[1];
  const bool late = (note[0] & 1) != 0;
  join();
  for (int s = NB * ngrp; s < npre; s += NB * ngrp) {
    fetch(s, npre, p.part_o, p.part_ml, chunk_row);
    join();
  }
  for (int s = 0; s < np; s += NB * ngrp) {
    fetch(s, np, p.own.part_o, p.own.part_ml, [&](int k) {
      return own_slot(p.own, J, wa + k, seq, np == 1, k == 0 && late) * p.own_rows + h0 - kRows * slice + qi;
    });
    join();
  }

  if (ngrp > 1) {
    __shared__ f32x4 so[256];
    __shared__ f32x2 sm[256];
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

template <typename T, int D, int DMA, int PG>
hipError_t launch(const PrefixParams& p, hipStream_t st) {
  const int own_wgs = PG > 0 ? (p.own.n_waves + 3) / 4 : p.own.n_waves;
  const dim3 grid((unsigned)(p.n_pre + own_wgs));
  if (grid.x > 0) {
    hipLaunchKernelGGL((pf_prefix_kernel<T, D, DMA, PG>), grid, dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((pf_prefix_merge_kernel<T, D>),
                     dim3((unsigned)(p.own.B * p.Hkv * ((p.g + p.merge_heads - 1) / p.merge_heads))), dim3(256), 0, st, p);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_pages(const PrefixParams& p, hipStream_t st) {
  if (!p.dma) return launch<T, D, 0, 0>(p, st);
  constexpr int PG = OwnGeo<T, D>::RPL == 8 ? 8 : 4;
  if (p.dma == 16) return p.thin ? launch<T, D, 16, 16>(p, st) : launch<T, D, 16, 0>(p, st);
  if (p.dma == 2) return p.thin ? launch<T, D, 2, kSplit>(p, st) : launch<T, D, 2, 0>(p, st);
  return p.thin ? launch<T, D, 1, PG>(p, st) : launch<T, D, 1, 0>(p, st);
}

template <typename T>
hipError_t launch_dim(const PrefixParams& p, int D, hipStream_t st) {
  if (D == 64) return launch_pages<T, 64>(p, st);
  if (D == 128) return launch_pages<T, 128>(p, st);
  if constexpr (sizeof(T) == 2)
    if (D == 256) return launch_pages<T, 256>(p, st);
  return hipErrorInvalidValue;
}

}  // namespace prefix
}  // namespace pf
