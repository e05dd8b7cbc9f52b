// Rotary positions with several axes (gfx950): q and k rotated into new
// tensors, or q rotated and k, v appended to a paged pool.
//
// Pair i of a row (elements i and i + D/2, rotate-half) belongs to one axis
// (time, height, width, ...): the first sections[0] pairs to axis 0, the next
// sections[1] to axis 1, and so on. With p the token's position on that axis,
// c1, c2, s1, s2 the table values cos[p][i], cos[p][i + D/2], sin[p][i],
// sin[p][i + D/2] and x1, x2 the pair:
//   forward   y1 = x1 c1 - x2 s1,  y2 = x2 c2 + x1 s2
//   inverse   y1 = x1 c1 + x2 s2,  y2 = x2 c2 - x1 s1   (the transpose: the VJP)
// in float32, rounded once to T.
// One axis is plain RoPE at arbitrary positions.
//
// Bound by memory: every element is read and written once. A thread owns E
// consecutive pairs of one token -- 16 bytes of each half where D / 2 allows --
// for NH heads: it looks the token's positions and table values up once (they
// come from the caches: neighbouring threads and heads share them) and then
// streams NH pairs of chunks. Inputs are read with their own strides, so the
// transposed views that a projection leaves are not copied first.
//
// A token with a position outside the tables gives zeros (and, appended,
// leaves the pool as it was): positions live in device memory and cannot be
// refused by the host.
#include "pf_common.hpp"
#include "pf_kernels.hpp"

#include <algorithm>

namespace pf {

namespace {

// E elements, element-aligned: rows need no 16-byte alignment.
template <typename T, int E>
struct Vec {
  typedef T type __attribute__((ext_vector_type(E), aligned(sizeof(T))));
};

template <int E>
__device__ inline void load_table(const float* t, float* out) {
  typedef typename Vec<float, E>::type v;
  const v x = *reinterpret_cast<const v*>(t);
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = x[e];
}

// Entry `which` of a parameter's three: by selects, as an indexed read would
// keep the parameters in scratch memory.
template <typename V>
__device__ inline V pick(const V (&v)[3], int which) {
  V x = v[0];
  if (which == 1) x = v[1];
  if (which == 2) x = v[2];
  return x;
}

// A token's table rows, one for each axis, in a vector (a struct or an array
// of them goes to LDS for the choices of row_of), and whether all of them lie
// inside the tables.
template <typename I>
__device__ inline i32x4 axis_rows(const RopeAxesParams& p, int b, int s, bool* inside) {
  static_assert(kMaxRopeAxes == 4, "four rows");
  const I* at = static_cast<const I*>(p.positions) + b * p.pos_stride[1] + s * p.pos_stride[2];
  const uint64_t n = p.rope_len;
  auto in = [&](I pos) { return (uint64_t)(int64_t)pos < n; };  // and not negative
  if (p.axes == 1) {
    const I x = at[0];
    *inside = in(x);
    return (i32x4){(int)x, 0, 0, 0};
  }
  // all four at once (those past the last axis repeat it), not one after another
  const int last = p.axes - 1;
  const I x0 = at[0], x1 = at[p.pos_stride[0]], x2 = at[min(2, last) * p.pos_stride[0]],
          x3 = at[last * p.pos_stride[0]];
  *inside = (bool)(in(x0) & in(x1) & in(x2) & in(x3));
  return (i32x4){(int)x0, (int)x1, (int)x2, (int)x3};
}
// The row of pair i. ends[a] is past every pair from the last axis on.
__device__ inline int row_of(const RopeAxesParams& p, const i32x4& rows, int i) {
  int r = rows[0];
  if (i >= p.ends[0]) r = rows[1];
  if (i >= p.ends[1]) r = rows[2];
  if (i >= p.ends[2]) r = rows[3];
  return r;
}

template <typename T, int E, bool NT>
__device__ inline typename Vec<T, E>::type get(const T* a) {
  typedef typename Vec<T, E>::type vT;
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const vT*>(a));
  else return *reinterpret_cast<const vT*>(a);
}
template <typename T, int E, bool NT>
__device__ inline void put(T* a, typename Vec<T, E>::type v) {
  typedef typename Vec<T, E>::type vT;
  if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<vT*>(a));
  else *reinterpret_cast<vT*>(a) = v;
}

template <typename T, int E, int NH, bool APPEND>
__global__ __launch_bounds__(256) void pf_rope_axes_kernel(RopeAxesParams p) {
  typedef typename Vec<T, E>::type vT;
  constexpr bool NT = NH > 1;
  const int half = p.D / 2;
  // blockIdx.y: the tensor (q, k, v) and its head group -- uniform, so that
  // bases and strides are scalars; x: (batch, token, chunk).
  int hg = blockIdx.y, which = 0;
  if (hg >= p.groups[0]) {
    hg -= p.groups[0];
    which = 1;
    if (APPEND && hg >= p.groups[1]) {
      hg -= p.groups[1];
      which = 2;
    }
  }
  const uint32_t item = blockIdx.x * 256u + threadIdx.x;
  if (item >= p.n_items) return;
  const uint32_t tok = fast_div(item, p.div_chunks);
  const int c = (int)(item - tok * p.div_chunks.d);
  const uint32_t bt = fast_div(tok, p.div_seq);
  const int b = (int)bt, s = p.s0 + (int)(tok - bt * p.div_seq.d);
  const int h0 = hg * NH, heads = pick(p.heads, which), nh = min(NH, heads - h0);
  const int i0 = c * E;  // the thread's first pair

  // Lookups first, the rows of x behind them: loads complete in order, so the
  // table loads that need the lookups wait for nothing else.
  bool live = true;
  int64_t own = 0;  // append: the token's position in its sequence
  i32x4 rows;
  bool inside;
  if constexpr (APPEND) {
    own = (int64_t)p.position[(int64_t)b * p.position_stride] + s;
    live = p.seq_lens == nullptr || s < p.seq_lens[b];
  }
  if (APPEND && p.positions == nullptr) {
    rows = (i32x4){(int)own, 0, 0, 0};
    inside = own >= 0 && own < p.rope_len;
  } else {
    rows = p.pos64 ? axis_rows<int64_t>(p, b, s, &inside) : axis_rows<int32_t>(p, b, s, &inside);
  }

  const int64_t sh = pick(p.sh, which);
  const T* src = static_cast<const T*>(pick(p.x, which)) + h0 * sh + b * pick(p.sb, which) + s * pick(p.ss, which) + i0;
  vT lo[NH], hi[NH];
  if (live) {
#pragma unroll
    for (int j = 0; j < NH; ++j)
      if (j < nh) {
        lo[j] = get<T, E, NT>(src + j * sh);
        hi[j] = get<T, E, NT>(src + j * sh + half);
      }
  }
  live = live && inside;

  // Where the rows go; pools: only where the position has a page.
  T* dst = nullptr;
  int64_t step = 0;  // from head to head
  if (!APPEND || which == 0) {
    dst = static_cast<T*>(pick(p.out, which)) + (((int64_t)b * heads + h0) * p.S + s) * p.D + i0;
    step = (int64_t)p.S * p.D;
  } else if (live && own >= 0) {
    // own < 2^31 wherever it has a page
    const uint32_t lp = (uint64_t)own >> 31 ? ~0u : fast_div((uint32_t)own, p.div_page);
    if (lp < (uint32_t)p.pages_per_seq) {
      const int page = p.block_tables[(int64_t)b * p.pages_per_seq + lp];
      const int off = (int)own - (int)lp * p.page_size;
      if (page >= 0 && page < p.num_pages) {
        dst = static_cast<T*>(pick(p.out, which)) +
              (((int64_t)page * heads + h0) * p.page_size + off) * p.D + i0;
        step = (int64_t)p.page_size * p.D;
      }
    }
  }
  if (dst == nullptr) return;

  if (APPEND && which == 2) {
#pragma unroll
    for (int j = 0; j < NH; ++j)
      if (j < nh) {
        put<T, E, NT>(dst + j * step, lo[j]);
        put<T, E, NT>(dst + j * step + half, hi[j]);
      }
    return;
  }
  if (!live) {
#pragma unroll
    for (int j = 0; j < NH; ++j)
      if (j < nh) {
        put<T, E, NT>(dst + j * step, (vT)(Elem<T>::from_f32(0.f)));
        put<T, E, NT>(dst + j * step + half, (vT)(Elem<T>::from_f32(0.f)));
      }
    return;
  }

  float c1[E], c2[E], s1[E], s2[E];
  const int row = row_of(p, rows, i0);
  bool cut = false;  // an axis ends inside the thread's pairs
#pragma unroll
  for (int a = 0; a < kMaxRopeAxes - 1; ++a) cut = cut || (i0 < p.ends[a] && p.ends[a] < i0 + E);
  if (!cut) {
    const float* cr = p.cos + (int64_t)row * p.D + i0;
    const float* sr = p.sin + (int64_t)row * p.D + i0;
    load_table<E>(cr, c1);
    load_table<E>(cr + half, c2);
    load_table<E>(sr, s1);
    load_table<E>(sr + half, s2);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t at = (int64_t)row_of(p, rows, i0 + e) * p.D + i0 + e;
      c1[e] = p.cos[at];
      c2[e] = p.cos[at + half];
      s1[e] = p.sin[at];
      s2[e] = p.sin[at + half];
    }
  }
  if (p.inverse) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = s1[e];
      s1[e] = -s2[e];
      s2[e] = -t;
    }
  }
#pragma unroll
  for (int j = 0; j < NH; ++j)
    if (j < nh) {
      vT y1, y2;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x1 = Elem<T>::to_f32(lo[j][e]), x2 = Elem<T>::to_f32(hi[j][e]);
        // the fused operand is fixed, so that every instance gives the same bits
        y1[e] = Elem<T>::from_f32(fmaf(x1, c1[e], -(x2 * s1[e])));
        y2[e] = Elem<T>::from_f32(fmaf(x2, c2[e], x1 * s2[e]));
      }
      put<T, E, NT>(dst + j * step, y1);
      put<T, E, NT>(dst + j * step + half, y2);
    }
}

template <typename T, int E, int NH, bool APPEND>
hipError_t launch_heads(RopeAxesParams p, hipStream_t st) {
  const int chunks = p.D / 2 / E;
  unsigned groups = 0;
  for (int w = 0; w < 3; ++w) {
    p.groups[w] = w < (APPEND ? 3 : 2) ? (p.heads[w] + NH - 1) / NH : 0;
    groups += p.groups[w];
  }
  p.div_chunks = fast_divisor(chunks);
  p.div_page = fast_divisor(APPEND ? p.page_size : 1);
  // 32-bit items: past 2^31 of them, the tokens in several launches.
  const int64_t most = (((int64_t)1 << 31) - 256) / ((int64_t)p.B * chunks);
  const int seq = p.S;
  for (int s0 = 0; s0 < seq; s0 += (int)std::min<int64_t>(most, seq)) {
    const int n = (int)std::min<int64_t>(most, seq - s0);
    p.s0 = s0;
    p.div_seq = fast_divisor(n);
    p.n_items = (uint32_t)((int64_t)p.B * n * chunks);
    hipLaunchKernelGGL((pf_rope_axes_kernel<T, E, NH, APPEND>), dim3((p.n_items + 255) / 256, groups), dim3(256), 0,
                       st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || n == seq - s0) return e;
  }
  return hipSuccess;
}

// Calls that move kStreamBytes or more run four heads a thread with
// non-temporal loads and stores, smaller ones a head a thread (as many waves as
// there can be) through the caches, where what reads the result next finds it.
// Only for whole 16-byte chunks. (Strided inputs, forward: 32768 tokens, 32 + 8
// float16 heads of 128, 671 MB: 170 us with a head a thread, 137 with four, 121
// = 5.8 TB/s with four and non-temporal; a float32 step of 37 MB a launch: 8.7,
// 9.0 and 10.1 us; 8 tokens: 3.0 and 3.4 us. On one shape the two forms cross at
// 40-60 MB.)
constexpr int64_t kStreamBytes = (int64_t)48 << 20;
template <typename T, int E, bool APPEND>
hipError_t launch_pairs(const RopeAxesParams& p, hipStream_t st) {
  if constexpr (E * sizeof(T) == 16) {
    const int64_t bytes =
        (int64_t)p.B * p.S * (p.heads[0] + p.heads[1] + (APPEND ? p.heads[2] : 0)) * p.D * 2 * (int)sizeof(T);
    if (bytes >= kStreamBytes) return launch_heads<T, E, 4, APPEND>(p, st);
  }
  return launch_heads<T, E, 1, APPEND>(p, st);
}

template <typename T, bool APPEND>
hipError_t launch_typed(const RopeAxesParams& p, hipStream_t st) {
  const int half = p.D / 2;
  if constexpr (sizeof(T) == 2)
    if (half % 8 == 0) return launch_pairs<T, 8, APPEND>(p, st);
  if (half % 4 == 0) return launch_pairs<T, 4, APPEND>(p, st);
  if (half % 2 == 0) return launch_pairs<T, 2, APPEND>(p, st);
  return launch_pairs<T, 1, APPEND>(p, st);
}

}  // namespace

hipError_t launch_rope_axes(const RopeAxesParams& p, int dtype, bool append, hipStream_t stream) {
  switch (dtype) {
    case kF32: return append ? launch_typed<float, true>(p, stream) : launch_typed<float, false>(p, stream);
    case kBF16: return append ? launch_typed<bf16_t, true>(p, stream) : launch_typed<bf16_t, false>(p, stream);
    case kF16: return append ? launch_typed<f16_t, true>(p, stream) : launch_typed<f16_t, false>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pf
