// !!! This is a file automatically generated by hipify!!!
#include "hip/hip_runtime.h"
// Group norm over channels-last activations, with the activation and the
// block's residual in the same pass. x is [N, HW, C], a group is C / G
// neighbouring channels of one sample, M = HW * C / G:
//
//   xh = (x - mean) / sqrt(var + eps)     z = gamma xh + beta (+ residual)
//   y  = act(z)
//   dz = dy act'(z)   dbeta = sum dz   dgamma = sum dz xh   dresidual = dz
//   dx = rstd (gamma dz - s1 - xh s2)
//   s1 = sum_group gamma dz / M   s2 = sum_group gamma dz xh / M
//
// A ReLU's gradient hangs on the sign of z alone. The forward pass leaves it
// as one bit a value (a byte for each vector), so that the backward pass reads
// neither the residual nor what makes z: 1/16 of a tensor for a whole one.
// Where fp32 does not tell the sign the forward pass takes z in 64 bits.
//
// Nothing here adds in an order that changes: every sum goes through slots
// of its own that are added in a fixed order.

#pragma once

#include "common.h"

#include <c10/core/DeviceGuard.h>

namespace eg {
namespace gn {

constexpr int BLOCK = 256, JOIN = 1024;
enum Act { NONE = 0, RELU = 1, SILU = 2 };
constexpr int RELU_BITS = 3;    // a ReLU that leaves its bits

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const Vec<T, V>& a) {
  *reinterpret_cast<Vec<T, V>*>(p) = a;
}

// Clears the values of g whose bit is not set.
template <typename T, int V>
__device__ __forceinline__ void keep(Vec<T, V>& g, unsigned bits) {
  if constexpr (sizeof(T) == 4) {
    auto* w = reinterpret_cast<unsigned*>(g.v);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] &= __builtin_amdgcn_sbfe(bits, j, 1);
  } else if constexpr (V > 1) {
    auto* w = reinterpret_cast<unsigned*>(g.v);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const unsigned low = __builtin_amdgcn_sbfe(bits, 2 * j, 1);
      const unsigned high = __builtin_amdgcn_sbfe(bits, 2 * j + 1, 1);
      w[j] &= __builtin_amdgcn_perm(high, low, 0x05040100);
    }
  } else if (!(bits & 1)) {
    g.v[0] = (T)0.f;
  }
}

__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));   // off by a step or two
}

// y of one vector, and with RELU_BITS a bit for each z that is not below or
// at zero. mean, scale and shift make z = (x - mean) scale + shift (+ r).
// `exact(j)` is the j-th z in 64 bits; it decides where a z is within the
// rounding of its terms of zero, `limit` being 2^-20 of those that do not
// change from value to value.
template <typename T, int V, int P, int ACT, typename Exact>
__device__ __forceinline__ unsigned activate(
    Vec<T, V>& a, const Vec<T, V>& b, bool res, const float (&mean)[P],
    const float (&scale)[V], const float (&shift)[V], float limit,
    Exact exact) {
  float z[V], least = 0x1p126f;
#pragma unroll
  for (int j = 0; j < V; ++j)
    z[j] = fmaf((float)a.v[j] - mean[P == 1 ? 0 : j], scale[j], shift[j]);
  if (res) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float r = (float)b.v[j];
      z[j] += r;
      if (ACT == RELU_BITS)
        least = fminf(least, fmaf(fabsf(r), -0x1p-19f, fabsf(z[j])));
    }
  } else if (ACT == RELU_BITS) {
#pragma unroll
    for (int j = 0; j < V; ++j) least = fminf(least, fabsf(z[j]));
  }
  unsigned bits = 0;
  if (ACT == RELU_BITS) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      bits |= (z[j] <= 0.f ? 0u : 1u) << j;    // NaN passes its gradient
    if (least <= limit) {
      bits = 0;
#pragma unroll 1
      for (int j = 0; j < V; ++j) bits |= (exact(j) <= 0.0 ? 0u : 1u) << j;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (ACT == RELU || ACT == RELU_BITS)
      z[j] = z[j] < 0.f ? 0.f : z[j];          // NaN stays NaN
    if (ACT == SILU) z[j] *= sigmoid(z[j]);
    a.v[j] = (T)z[j];
  }
  return bits;
}

// How the [HW, C] rows of a sample are dealt out: a block takes one chunk of
// rows (blockIdx.x counts samples, then chunks) and one tile of columns
// (blockIdx.z); a thread keeps one column of V channels and takes every
// `rows`-th row of the chunk.
struct Deal {
  int hw, c, cols, lanes, rows, per_chunk, chunks;
};

struct Place {
  int n, chunk, begin, count;   // the chunk's first row and its rows
  int lane, r, col;             // column within the tile, row offset, column
  bool on;
  __device__ __forceinline__ explicit Place(const Deal& d) {
    n = blockIdx.x / d.chunks;
    chunk = blockIdx.x % d.chunks;
    begin = chunk * d.per_chunk;
    count = min(d.per_chunk, d.hw - begin);
    lane = threadIdx.x % d.lanes;
    r = threadIdx.x / d.lanes;
    col = blockIdx.z * d.lanes + lane;
    on = r < d.rows && col < d.cols;
  }
};

// Adds K values over the rows of a block, column by column, in a fixed order;
// the sums are those of the threads with r == 0. slot: BLOCK / 2 * K floats.
template <int K>
__device__ __forceinline__ void add_rows(float (&v)[K], float* slot, int r,
                                         int lane, int lanes, int rows) {
  for (int live = rows; live > 1;) {
    const int half = (live + 1) / 2;
    if (r >= half && r < live) {
#pragma unroll
      for (int j = 0; j < K; ++j)
        slot[((r - half) * lanes + lane) * K + j] = v[j];
    }
    __syncthreads();
    if (r < live - half) {
#pragma unroll
      for (int j = 0; j < K; ++j) v[j] += slot[(r * lanes + lane) * K + j];
    }
    __syncthreads();
    live = half;
  }
}

struct Pair {
  float a, b;
  __device__ __forceinline__ Pair& operator+=(const Pair& o) {
    a += o.a;
    b += o.b;
    return *this;
  }
};

__device__ __forceinline__ Pair across(const Pair& p, int m) {
  return {__shfl_xor(p.a, m), __shfl_xor(p.b, m)};
}

__device__ __forceinline__ double across(double v, int m) {
  return __shfl_xor(v, m);
}

// the sum of a block's values, in every thread
template <typename F>
__device__ __forceinline__ F add_block(F v, F* slot) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  F s = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) s += slot[w];
  return s;
}

// ---- one block a slab ----------------------------------------------------
//
// A slab is all rows of one sample in a slice of whole groups. Where it fits
// into a block's registers (I vectors of 16 bytes a thread) it is read once:
// statistics are taken from the registers, and what is written comes out of
// them too.

constexpr int SLAB = 512;   // threads at most, and groups of a slice
constexpr int FWD_VECTORS = 16, BWD_VECTORS = 8;   // of a thread, at most

struct Slab {
  int hw, c, lanes, rows, slices;   // lanes: columns of a slice
  int groups, cpg, in_slice, per;   // groups of the sample and of a slice;
                                    // per: threads that add one group up
};

struct Spot {
  int n, lane, r, first;            // first: the slice's first channel
  bool on;
  __device__ __forceinline__ Spot(const Slab& d, int v) {
    // blocks go round the 8 XCDs in turn; slices of one sample share cache
    // lines, so each XCD is given a run of neighbours
    const unsigned all = gridDim.x, b = blockIdx.x;
    const unsigned x = b & 7u, q = all >> 3, rest = all & 7u;
    const unsigned at = x * q + min(x, rest) + (b >> 3);
    n = at / d.slices;
    first = (int)(at % d.slices) * d.lanes * v;
    lane = threadIdx.x % d.lanes;
    r = threadIdx.x / d.lanes;
    on = r < d.rows;
  }
};

// Adds each group's entries of a table [rows, width] in LDS, width being
// in_slice groups of `w`, and hands the sum to `done` in one thread a group.
template <typename S, typename E, typename Done>
__device__ __forceinline__ void add_groups(const E* table, int rows, int w,
                                           const Slab& d, Done done) {
  const int j = threadIdx.x % d.per;
  const int width = w * d.in_slice;
  const int down = d.per / w, right = d.per % w;
  for (int q = threadIdx.x / d.per; q < d.in_slice;
       q += blockDim.x / d.per) {
    S s{};
    int row = j / w, col = j % w;
    while (row < rows) {
      s += table[row * width + q * w + col];
      row += down;
      col += right;
      if (col >= w) {
        col -= w;
        ++row;
      }
    }
    for (int m = d.per / 2; m; m >>= 1) s += across(s, m);
    if (j == 0) done(q, s);
  }
}

// ---- host -----------------------------------------------------------------

static Deal deal(long hw, int c, int v, long n) {
  Deal d;
  d.hw = (int)hw;
  d.c = c;
  d.cols = c / v;
  d.lanes = std::min(d.cols, BLOCK);
  d.rows = BLOCK / d.lanes;
  const long tiles = (d.cols + d.lanes - 1) / d.lanes;
  // About 2,048 blocks, eight a CU, and no chunk under sixteen rows a thread:
  // its sums cost as much as some rows. On 4x128x128x320 forward and backward
  // 4 rows a thread took 108 us, 16 take 103; on 1x512x512x128 512 blocks
  // took 58 us, 2,048 take 46 and 4,096 took 55.
  const long wanted = std::max<long>(1, 2048 / std::max<long>(1, n * tiles));
  const long most = std::max<long>(1, hw / (16L * d.rows));
  const long chunks = std::min(wanted, most);
  d.per_chunk = (int)((hw + chunks - 1) / chunks);
  d.chunks = (int)((hw + d.per_chunk - 1) / d.per_chunk);
  return d;
}

struct Shape {
  long n, hw;
  int c, groups, cpg;
};

static Shape shape_of(const torch::Tensor& x, const torch::Tensor& gamma,
                      const torch::Tensor& beta, long groups, long act,
                      const c10::optional<torch::Tensor>& res) {
  CHECK_IN(x);
  TORCH_CHECK(x.dim() == 4, "group_norm takes [N, H, W, C], got ", x.dim(),
              " dimensions");
  const auto t = x.scalar_type();
  TORCH_CHECK(t == torch::kBFloat16 || t == torch::kHalf ||
                  t == torch::kFloat32,
              "group_norm takes bf16, fp16 or fp32, got ", t);
  Shape s;
  s.n = x.size(0);
  s.hw = x.size(1) * x.size(2);
  const long c = x.size(3);
  TORCH_CHECK(s.hw < (1L << 31) && c < (1L << 24), "group_norm: a sample of ",
              s.hw, " x ", c, " is too large");
  TORCH_CHECK(s.n < (1L << 23), "group_norm: a batch of ", s.n,
              " is too large");
  TORCH_CHECK(groups > 0 && c > 0 && c % groups == 0, "group_norm: ", c,
              " channels do not divide into ", groups, " groups");
  TORCH_CHECK(act >= NONE && act <= SILU, "group_norm: no activation ", act);
  s.c = (int)c;
  s.groups = (int)groups;
  s.cpg = (int)(c / groups);
  auto vec = [&](const torch::Tensor& p, const char* name) {
    TORCH_CHECK(p.device() == x.device(), "group_norm: ", name,
                " must be on x's GPU");
    TORCH_CHECK(p.scalar_type() == torch::kFloat32 && p.is_contiguous() &&
                    p.dim() == 1 && p.numel() == c,
                "group_norm: ", name, " must be a contiguous fp32 vector of ",
                c);
  };
  vec(gamma, "gamma");
  vec(beta, "beta");
  if (res) {
    TORCH_CHECK(res->device() == x.device() && res->scalar_type() == t &&
                    res->sizes() == x.sizes() && res->is_contiguous(),
                "group_norm: the residual must be like x, and contiguous");
  }
  return s;
}

// the widest vector, up to 16 bytes, that the channels and every pointer
// divide into
static int width(const Shape& s, int size,
                 std::initializer_list<const void*> ptrs) {
  uintptr_t bits = 0;
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
  int v = 16 / size;
  while (v > 1 && (s.c % v || bits % (v * size))) v /= size == 4 ? 4 : 2;
  if (size == 2 && v == 4) v = 2;
  return v;
}

template <typename T, int V>
struct Tag {
  using type = T;
  static constexpr int v = V;
};

// calls f with the element type and the vector width as types
template <typename F>
static void with_type(c10::ScalarType t, int v, F f) {
  auto two = [&](auto zero) {
    using T = decltype(zero);
    if (v == 8) f(Tag<T, 8>());
    else if (v == 2) f(Tag<T, 2>());
    else f(Tag<T, 1>());
  };
  if (t == torch::kBFloat16) two((__bf16)0.f);
  else if (t == torch::kHalf) two((_Float16)0.f);
  else if (v == 4) f(Tag<float, 4>());
  else f(Tag<float, 1>());
}

template <typename T, int V, int I, int P>
struct SlabTag : Tag<T, V> {
  static constexpr int i = I, p = P;
};

// calls f with the types of a slab kernel: I is the least of 1, 2, 4, 8 and
// 16 that holds `vectors` (with narrow vectors of 4 and 16, which are rare)
template <typename F>
static void with_slab(c10::ScalarType t, int v, int vectors, bool whole,
                      F f) {
  with_type(t, v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    constexpr bool full = V * sizeof(T) == 16;
    auto pick = [&](auto parts) {
      constexpr int P = decltype(parts)::v;
      if (full && vectors == 1) f(SlabTag<T, V, full ? 1 : 4, P>());
      else if (full && vectors == 2) f(SlabTag<T, V, full ? 2 : 4, P>());
      else if (vectors <= 4) f(SlabTag<T, V, 4, P>());
      else if (vectors <= 8) f(SlabTag<T, V, 8, P>());
      else f(SlabTag<T, V, 16, P>());
    };
    if (whole) pick(Tag<T, 1>());
    else pick(Tag<T, V>());
  });
}

// calls f with the activation as a type
template <typename F>
static void with_act(long act, bool bits, F f) {
  if (act == RELU && bits) f(Tag<int, RELU_BITS>());
  else if (act == RELU) f(Tag<int, RELU>());
  else if (act == SILU) f(Tag<int, SILU>());
  else f(Tag<int, NONE>());
}

// How a sample is cut into slabs of at most `most` vectors a thread; threads
// is 0 where even the narrowest slice is more than that.
struct Cut {
  Slab d;
  int threads, vectors;
};

static Cut cut(const Shape& s, int v, int size, int most) {
  Cut out{};
  auto gcd = [](int a, int b) {
    while (b) {
      const int t = a % b;
      a = b;
      b = t;
    }
    return a;
  };
  // the narrowest slice has whole groups and whole vectors
  const int base = s.cpg / gcd(s.cpg, v), cols = s.c / v, units = cols / base;
  auto fits = [&](int k) {
    const long lanes = (long)base * k;
    return lanes <= SLAB && lanes * v <= (long)SLAB * s.cpg &&
           (s.hw + SLAB / lanes - 1) / (SLAB / lanes) <= most;
  };
  if (!fits(1)) return out;
  // Wider while a row of the slice is under a cache line, or while a block
  // has under 1,024 vectors and there are blocks to spare (two a CU).
  int best = 1;
  for (int k = 2; k <= units && fits(k); ++k) {
    if (units % k) continue;
    const bool narrow = (long)base * best * v * size < 64;
    const bool small = (long)base * best * s.hw < 1024 &&
                       s.n * (units / k) >= 512;
    if (!narrow && !small) break;
    best = k;
  }
  Slab& d = out.d;
  d.hw = (int)s.hw;
  d.c = s.c;
  d.lanes = base * best;
  d.slices = units / best;
  d.groups = s.groups;
  d.cpg = s.cpg;
  d.in_slice = d.lanes * v / s.cpg;
  const long want = ((long)d.lanes * s.hw + 63) / 64 * 64;
  out.threads = (int)std::min<long>(SLAB, std::max<long>(64, want));
  d.rows = out.threads / d.lanes;
  const long need = (s.hw + d.rows - 1) / d.rows;
  out.vectors = 1;
  while (out.vectors < need) out.vectors *= 2;
  d.per = 1;
  while (d.per < 64 && 2 * d.per * d.in_slice <= out.threads) d.per *= 2;
  return out;
}

}  // namespace gn
}  // namespace eg
