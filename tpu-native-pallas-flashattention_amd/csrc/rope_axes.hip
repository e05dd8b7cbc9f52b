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

namespace pf {

namespace {

// a / b and a % b for a >= 0, in 32 bits where they do (a 64-bit division is
// several hundred instructions).
__device__ inline int64_t divmod(int64_t a, int b, int* rem) {
  if (((uint64_t)a >> 32) == 0) {
    const uint32_t q = (uint32_t)a / (uint32_t)b;
    *rem = (int)((uint32_t)a - q * (uint32_t)b);
    return q;
  }
  const int64_t q = a / b;
  *rem = (int)(a - q * b);
  return q;
}

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

__device__ inline int64_t position(const RopeAxesParams& p, int axis, int b, int s) {
  const int64_t at = axis * p.pos_stride[0] + b * p.pos_stride[1] + s * p.pos_stride[2];
  return p.pos64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
}

template <typename T, int E, int NH, bool APPEND>
__global__ __launch_bounds__(256) void pf_rope_axes_kernel(RopeAxesParams p, int64_t n_items) {
  typedef typename Vec<T, E>::type vT;
  const int half = p.D / 2, HC = half / E;
  int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (it >= n_items) return;
  int c, s, hg;
  it = divmod(it, HC, &c);
  it = divmod(it, p.S, &s);
  const int n_grp[3] = {(p.heads[0] + NH - 1) / NH, (p.heads[1] + NH - 1) / NH, APPEND ? (p.heads[2] + NH - 1) / NH : 0};
  const int b = (int)divmod(it, n_grp[0] + n_grp[1] + n_grp[2], &hg);
  int which = 0;  // q, k, v
  if (hg >= n_grp[0]) {
    hg -= n_grp[0];
    which = 1;
    if (APPEND && hg >= n_grp[1]) {
      hg -= n_grp[1];
      which = 2;
    }
  }
  const int h0 = hg * NH, heads = p.heads[which], nh = min(NH, heads - h0);
  const int i0 = c * E;  // the thread's first pair

  bool live = true;
  int64_t own = 0;  // append: the token's position in its sequence
  if constexpr (APPEND) {
    live = p.seq_lens == nullptr || s < p.seq_lens[b];
    own = (int64_t)p.position[(int64_t)b * p.position_stride] + s;
  }
  // The input does not depend on the lookups: under way beside them.
  const T* src = static_cast<const T*>(p.x[which]) + b * p.sb[which] + h0 * p.sh[which] + s * p.ss[which] + i0;
  vT lo[NH], hi[NH];
  if (live) {
#pragma unroll
    for (int j = 0; j < NH; ++j)
      if (j < nh) {
        lo[j] = __builtin_nontemporal_load(reinterpret_cast<const vT*>(src + j * p.sh[which]));
        hi[j] = __builtin_nontemporal_load(reinterpret_cast<const vT*>(src + j * p.sh[which] + half));
      }
  }

  // The table rows of the first and last pair's axis; ends[] covers all pairs.
  int64_t row0 = own, row1 = own;
  int a0 = 0, a1 = 0;
  if (live) {
    if (!APPEND || p.positions != nullptr) {
#pragma unroll
      for (int a = 0; a < kMaxRopeAxes; ++a) {
        if (a >= p.axes) break;
        const int64_t pos = position(p, a, b, s);
        live = live && pos >= 0 && pos < p.rope_len;
        if (a == 0 || i0 >= p.ends[a - 1]) {
          row0 = pos;
          a0 = a;
        }
        if (a == 0 || i0 + E - 1 >= p.ends[a - 1]) {
          row1 = pos;
          a1 = a;
        }
      }
    } else {
      live = own >= 0 && own < p.rope_len;
    }
  }

  // Where the rows go; pools: only where the position has a page.
  T* dst = nullptr;
  int64_t step = 0;  // from head to head
  if (!APPEND || which == 0) {
    dst = static_cast<T*>(p.out[which]) + (((int64_t)b * heads + h0) * p.S + s) * p.D + i0;
    step = (int64_t)p.S * p.D;
  } else if (live && own >= 0) {
    int off;
    const int64_t lp = divmod(own, p.page_size, &off);
    if (lp < p.pages_per_seq) {
      const int page = p.block_tables[(int64_t)b * p.pages_per_seq + lp];
      if (page >= 0 && page < p.num_pages) {
        dst = static_cast<T*>(p.out[which]) +
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
        *reinterpret_cast<vT*>(dst + j * step) = lo[j];
        *reinterpret_cast<vT*>(dst + j * step + half) = hi[j];
      }
    return;
  }
  if (!live) {
#pragma unroll
    for (int j = 0; j < NH; ++j)
      if (j < nh) {
        *reinterpret_cast<vT*>(dst + j * step) = (vT)(Elem<T>::from_f32(0.f));
        *reinterpret_cast<vT*>(dst + j * step + half) = (vT)(Elem<T>::from_f32(0.f));
      }
    return;
  }

  float c1[E], c2[E], s1[E], s2[E];
  if (a0 == a1) {
    const float* cr = p.cos + row0 * p.D + i0;
    const float* sr = p.sin + row0 * p.D + i0;
    load_table<E>(cr, c1);
    load_table<E>(cr + half, c2);
    load_table<E>(sr, s1);
    load_table<E>(sr + half, s2);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      int64_t row = row0;
      if (i0 + e >= p.ends[a1 - 1]) row = row1;
      else if (a1 > a0 + 1 && i0 + e >= p.ends[a0]) {  // an axis that lies inside the thread's pairs
        int a = a0 + 1;
        while (i0 + e >= p.ends[a]) ++a;
        row = position(p, a, b, s);
      }
      const float* cr = p.cos + row * p.D + i0 + e;
      const float* sr = p.sin + row * p.D + i0 + e;
      c1[e] = cr[0];
      c2[e] = cr[half];
      s1[e] = sr[0];
      s2[e] = sr[half];
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
      *reinterpret_cast<vT*>(dst + j * step) = y1;
      *reinterpret_cast<vT*>(dst + j * step + half) = y2;
    }
}

template <typename T, int E, int NH, bool APPEND>
hipError_t launch_heads(const RopeAxesParams& p, hipStream_t st) {
  int64_t grps = 0;
  for (int w = 0; w < (APPEND ? 3 : 2); ++w) grps += (p.heads[w] + NH - 1) / NH;
  const int64_t n = (int64_t)p.B * p.S * grps * (p.D / 2 / E);
  const int64_t grid = (n + 255) / 256;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((pf_rope_axes_kernel<T, E, NH, APPEND>), dim3((unsigned)grid), dim3(256), 0, st, p, n);
  return hipGetLastError();
}

template <typename T, int E, bool APPEND>
hipError_t launch_pairs(const RopeAxesParams& p, hipStream_t st) {
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
