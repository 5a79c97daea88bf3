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

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>

namespace eg {
namespace gn {

constexpr int BLOCK = 256, JOIN = 1024;
enum Act { NONE = 0, RELU = 1, SILU = 2 };
constexpr int RELU_BITS = 3;    // a ReLU that leaves its bits

// V values as they lie in memory, two 16-bit ones to a word. They stay so
// until they are worked on: taken apart when they are loaded they would hold
// twice the registers, and the backward slab's blocks be one a CU for two.
template <typename T, int V>
struct Vec {
  static constexpr int BYTES = sizeof(T) * V;
  static constexpr int WORDS = BYTES < 4 ? 1 : BYTES / 4;
  unsigned w[WORDS];

  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else if constexpr (std::is_same_v<T, __bf16>) {
      return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    } else {
      const unsigned short h = (unsigned short)(w[j / 2] >> (j & 1 ? 16 : 0));
      return (float)__builtin_bit_cast(T, h);
    }
  }

  __device__ __forceinline__ void put(const float (&z)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = __float_as_uint(z[j]);
    } else if constexpr (V == 1) {
      w[0] = __builtin_bit_cast(unsigned short, (T)z[0]);
    } else {
      typedef T Two __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int j = 0; j < V / 2; ++j)
        w[j] = __builtin_bit_cast(unsigned,
                                  Two{(T)z[2 * j], (T)z[2 * j + 1]});
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
  Vec<T, V> a;
  if constexpr (Vec<T, V>::BYTES == 16) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    a.w[0] = t.x;
    a.w[1] = t.y;
    a.w[2] = t.z;
    a.w[3] = t.w;
  } else if constexpr (Vec<T, V>::BYTES == 4) {
    a.w[0] = *reinterpret_cast<const unsigned*>(p);
  } else {
    a.w[0] = *reinterpret_cast<const unsigned short*>(p);
  }
  return a;
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const Vec<T, V>& a) {
  if constexpr (Vec<T, V>::BYTES == 16)
    *reinterpret_cast<uint4*>(p) = make_uint4(a.w[0], a.w[1], a.w[2], a.w[3]);
  else if constexpr (Vec<T, V>::BYTES == 4)
    *reinterpret_cast<unsigned*>(p) = a.w[0];
  else
    *reinterpret_cast<unsigned short*>(p) = (unsigned short)a.w[0];
}

// Makes the compiler take a vector as new: between two passes over registers
// it would else keep what it made of each value in the first, in fp32.
template <typename T, int V>
__device__ __forceinline__ void renew(Vec<T, V>& a) {
#pragma unroll
  for (auto& w : a.w) asm volatile("" : "+v"(w));
}

// Clears the values of g whose bit is not set.
template <typename T, int V>
__device__ __forceinline__ void keep(Vec<T, V>& g, unsigned bits) {
#pragma unroll
  for (int j = 0; j < Vec<T, V>::WORDS; ++j) {
    if constexpr (sizeof(T) == 4 || V == 1) {
      g.w[j] &= __builtin_amdgcn_sbfe(bits, j, 1);
    } else {
      const unsigned low = __builtin_amdgcn_sbfe(bits, 2 * j, 1);
      const unsigned high = __builtin_amdgcn_sbfe(bits, 2 * j + 1, 1);
      g.w[j] &= __builtin_amdgcn_perm(high, low, 0x05040100);
    }
  }
}

// 1 / (1 + e^-z), off by a few steps; at both ends e^-z leaves the range of
// floats and the result is 0 or 1
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(
      1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

// y of one vector, and with RELU_BITS a bit for each z that is not below or
// at zero. mean, scale and shift make z = (x - mean) scale + shift (+ r); what
// a mean of 64 bits was rounded by is in the shift.
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
    z[j] = fmaf(a[j] - mean[P == 1 ? 0 : j], scale[j], shift[j]);
  if (res) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float r = b[j];
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
  }
  a.put(z);
  return bits;
}

struct Pair {
  float a, b;
  __device__ __forceinline__ Pair& operator+=(const Pair& o) {
    a += o.a;
    b += o.b;
    return *this;
  }
};

struct Twice {
  double a, b;
  __device__ __forceinline__ Twice& operator+=(const Twice& o) {
    a += o.a;
    b += o.b;
    return *this;
  }
};

// The value of the lane whose number differs in bit M, where lanes that differ
// in lower bits alone have the same: crossing within a row of 16 lanes is part
// of an instruction, and rows are swapped by one.
template <int M>
__device__ __forceinline__ unsigned other(unsigned v) {
  if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else if constexpr (M == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  } else {
    constexpr int ctrl = M == 1 ? 0xb1 : M == 2 ? 0x4e : M == 4 ? 0x141 : 0x140;
    return __builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, false);
  }
}

template <int M, typename S>
__device__ __forceinline__ S across(const S& v) {
  unsigned w[sizeof(S) / 4];
  __builtin_memcpy(w, &v, sizeof(S));
#pragma unroll
  for (unsigned i = 0; i < sizeof(S) / 4; ++i) w[i] = other<M>(w[i]);
  S o;
  __builtin_memcpy(&o, w, sizeof(S));
  return o;
}

// the sum over `per` neighbouring lanes, a power of two, in each of them
template <typename S>
__device__ __forceinline__ S add_lanes(S v, int per) {
  if (per > 1) v += across<1>(v);
  if (per > 2) v += across<2>(v);
  if (per > 4) v += across<4>(v);
  if (per > 8) v += across<8>(v);
  if (per > 16) v += across<16>(v);
  if (per > 32) v += across<32>(v);
  return v;
}

// the sum of a block's values, in every thread
template <typename F>
__device__ __forceinline__ F add_block(F v, F* slot) {
  v = add_lanes(v, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  F s = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) s += slot[w];
  return s;
}

// ---- slabs ----------------------------------------------------------------
//
// A slab is a chunk of one sample's rows in a slice of whole groups. Where all
// rows fit into a block's registers, I vectors of 16 bytes a thread, everything is made of one reading: statistics are taken
// from the registers, and what is written comes out of them too. Longer
// samples are read chunk by chunk for their sums, which a second kernel joins
// and a third applies.

constexpr int SLAB = 1024;  // threads at most
constexpr int SPAN = 512;   // threads that a slab is made for
constexpr int CHUNK_ROWS = 16;     // of a thread, where samples are longer
constexpr int WIDE_VECTORS = 4;    // of a thread, where there are more
constexpr int FWD_VECTORS = 16, BWD_VECTORS = 8;   // of a thread, at most

// threads at most in the forward pass, where each has P sums of 64 bits in LDS
constexpr int fwd_threads(int parts) { return parts > 4 ? SPAN : SLAB; }

// Divisions by what a launch fixes. An integer division is a chain of some 30
// instructions, and the few of a slab's plan took as long as its first loads.
struct Div {
  unsigned by, mul, shift;
  __device__ __forceinline__ unsigned of(unsigned n) const {   // n < 2^31
    return (__umulhi(n, mul) + n) >> shift;
  }
};

static Div div_by(unsigned by) {
  unsigned shift = 0;
  while ((1u << shift) < by) ++shift;
  const unsigned long one = 1UL << 32;
  return {by, (unsigned)(one * ((1UL << shift) - by) / by + 1), shift};
}

struct Slab {
  int hw, c, lanes, rows;           // lanes: columns of a slice
  int slices, chunks, per_chunk;    // of a sample; rows of a chunk
  int groups, cpg, in_slice;        // groups of the sample and of a slice
  Div by_lanes, by_rows, by_slices, by_chunks, by_subs, by_cpg;
  // adding a group up: threads for each, entries of a row, and how a thread
  // goes from one of its entries to the next
  int per, shift, w, down, right;
  Div by_w;
  // adding rows up, eight into one: rows that are left, entries, their shares
  struct { int to, n, step; Div by_n; } level[4];
  double inv;                       // 1 / values of a group of a sample
  // a slice is one of `subs` in a unit of `span` columns: the sample's, or a
  // group's where that alone is too wide
  int subs, span;
};

struct Spot {
  int n, chunk, slice, lane, r, first;   // first: the thread's first channel
  int begin, count;                      // the chunk's rows
  // Where a thread's row k is: at base + k * step + off. All but off is the
  // same for a whole block and stays in scalar registers, and off is 32 bits
  // of bytes, so that one register of a thread addresses all that it loads
  // and stores.
  long base, step;
  unsigned off;
  bool on;
  __device__ __forceinline__ Spot(const Slab& d, int v) {
    // blocks go round the 8 XCDs in turn; slices of one sample share cache
    // lines, so each XCD is given a run of neighbours
    const unsigned all = gridDim.x, b = blockIdx.x;
    const unsigned x = b & 7u, q = all >> 3, rest = all & 7u;
    const unsigned at = x * q + min(x, rest) + (b >> 3);
    const unsigned row = d.by_slices.of(at);
    slice = at - row * d.slices;
    n = d.by_chunks.of(row);
    chunk = row - n * d.chunks;
    begin = chunk * d.per_chunk;
    count = min(d.per_chunk, d.hw - begin);
    r = d.by_lanes.of(threadIdx.x);
    lane = threadIdx.x - r * d.lanes;
    const int unit = d.by_subs.of(slice);
    const int col = (slice - unit * d.subs) * d.lanes + lane;
    on = r < d.rows && col < d.span;
    const int c0 = (unit * d.span + col - lane) * v;
    first = on ? c0 + lane * v : 0;
    base = ((long)n * d.hw + begin) * d.c + c0;
    step = (long)d.rows * d.c;
    off = (unsigned)r * d.c + lane * v;
  }
  __device__ __forceinline__ bool has(int k, const Slab& d) const {
    return on && r + k * d.rows < count;
  }
  template <typename T>
  __device__ __forceinline__ T* row(T* p, int k) const {
    using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
    return reinterpret_cast<T*>(reinterpret_cast<Byte*>(p + base + k * step) +
                                (size_t)(off * (unsigned)sizeof(T)));
  }
  template <int V, typename T>
  __device__ __forceinline__ T* bits(T* p, int k) const {
    return p + (base + k * step) / V + (size_t)(off / V);
  }
};

// Calls f(k) for a thread's rows of a chunk: all but the last without asking
// for each whether it is there, so that the loads of U go out together.
template <int U, typename F>
__device__ __forceinline__ void each_row(const Spot& at, const Slab& d, F f) {
  if (!at.on) return;
  const int whole = d.by_rows.of(at.count);
  int k = 0;
  for (; k + U <= whole; k += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) f(k + u);
  }
  for (; k < whole; ++k) f(k);
  if (at.r + whole * d.rows < at.count) f(whole);
}

// Calls f(j, q) for a vector's parts with the place q of each in its slice's
// groups: one part, or a channel each.
template <int P, typename F>
__device__ __forceinline__ void each_part(int channel, const Slab& d, F f) {
  int q = d.by_cpg.of(channel), rest = channel - q * d.cpg;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    f(j, q);
    if (++rest == d.cpg) {
      rest = 0;
      ++q;
    }
  }
}

// Tables in LDS: K sums of each thread, one behind the other for all threads
// (so that neighbours write to neighbouring banks), [K][blockDim], a thread
// being r * lanes + lane.

// Adds the rows r of a table, eight into one at a time, in place, until at
// most `most` are left; their number is returned.
template <int K, typename F>
__device__ __forceinline__ int fold(F* table, const Slab& d, int most) {
  int rows = d.rows;
#pragma unroll 1
  for (int l = 0; rows > most; ++l) {
    // n threads for each of as many sums as there are threads for
    const int n = d.level[l].n, step = d.level[l].step;
    const int all = rows * d.lanes;
    const int at = d.level[l].by_n.of(threadIdx.x);
    for (int t = threadIdx.x - at * n; t < n; t += blockDim.x) {
      if (at >= step) break;
      for (int k = at; k < K; k += step) {
        F* e = table + k * blockDim.x + t;
        F s = e[0];
#pragma unroll
        for (int i = 1; i < 8; ++i)
          if (t + i * n < all) s += e[i * n];
        e[0] = s;
      }
    }
    __syncthreads();
    rows = d.level[l].to;
  }
  return rows;
}

// Adds each group's entries of the first `rows` rows of a table and hands the
// sum to `done` in one thread a group.
// get(e, row) is the row's e-th entry, counted through the slice's groups.
template <typename S, typename Get, typename Done>
__device__ __forceinline__ void add_groups(int rows, const Slab& d, Get get,
                                           Done done) {
  const int j = threadIdx.x & (d.per - 1);
  const int row0 = d.by_w.of(j), col0 = j - row0 * d.w;
  for (int q = threadIdx.x >> d.shift; q < d.in_slice;
       q += blockDim.x >> d.shift) {
    S s{};
    int row = row0, col = col0;
    while (row < rows) {
      s += get(q * d.w + col, row);
      row += d.down;
      col += d.right;
      if (col >= d.w) {
        col -= d.w;
        ++row;
      }
    }
    s = add_lanes(s, d.per);
    if (j == 0) done(q, s);
  }
}

// the e-th entry of a row, where a thread's K = P sums are a vector's parts
template <int P>
__device__ __forceinline__ double part(const double* table, const Slab& d,
                                       int e, int row) {
  return P == 1 ? table[row * d.lanes + e]
                : table[e % P * blockDim.x + row * d.lanes + e / P];
}

// The means and the sums of squared distances from them of a slab's groups,
// from the registers. emit(q, mean, m2) is called in one thread a group, with
// the means in mean_of. P: parts of a vector that have a mean each, 1 where it
// lies within a group. Sums of a vector's values, or of a channel's in one
// thread, are taken in fp32 and everything beyond in 64 bits. EXACT: all sums,
// the distances and their squares are in 64 bits: a ReLU's bits hang on the
// mean and rstd as much as on z.
// (With a thread's sums in fp32 these were 1e-8 off, and one in some 20 passes
// over the 16.8 M values of 256x32x32x64 had a bit wrong. It costs 0.7 us of
// 10.7 on 100x32x32x64 and 1.4 of 27.9 on 256x32x32x64 with its residual.)
template <typename T, int V, int I, int P, bool EXACT, typename Emit>
__device__ __forceinline__ void statistics(Vec<T, V> (&a)[I],
                                           const Spot& at, const Slab& d,
                                           double* table, double* mean_of,
                                           float (&mean)[P], Emit emit) {
  const int most = P == 1 ? SLAB : 8;    // as they are, or eight rows
  using Sum = std::conditional_t<P == 1 || EXACT, double, float>;
  Sum s[P] = {};
  auto get = [&](int e, int row) { return part<P>(table, d, e, row); };
#pragma unroll
  for (int k = 0; k < I; ++k) {
    if (at.has(k, d)) {
      if constexpr (P > 1 || EXACT) {
#pragma unroll
        for (int j = 0; j < V; ++j) s[P == 1 ? 0 : j] += a[k][j];
      } else {
        float t = a[k][0];
#pragma unroll
        for (int j = 1; j < V; ++j) t += a[k][j];
        s[0] += t;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j) table[j * blockDim.x + threadIdx.x] = s[j];
  __syncthreads();
  add_groups<double>(fold<P>(table, d, most), d, get,
                     [&](int q, double t) { mean_of[q] = t * d.inv; });
  __syncthreads();
  double mid[P];
  each_part<P>(at.lane * V, d, [&](int j, int q) {
    mid[j] = mean_of[q];
    mean[j] = (float)mid[j];
    s[j] = 0;
  });
#pragma unroll
  for (int k = 0; k < I; ++k) {
    renew<T, V>(a[k]);
    if (at.has(k, d)) {
      if constexpr (EXACT) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int p = P == 1 ? 0 : j;
          const double e = a[k][j] - mid[p];
          s[p] = fma(e, e, s[p]);
        }
      } else {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float e = a[k][j] - mean[P == 1 ? 0 : j];
          if (P == 1) t = fmaf(e, e, t);
          else s[j] = fmaf(e, e, (float)s[j]);
        }
        if (P == 1) s[0] += t;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j) table[j * blockDim.x + threadIdx.x] = s[j];
  __syncthreads();
  add_groups<double>(fold<P>(table, d, most), d, get,
                     [&](int q, double t) { emit(q, mean_of[q], t); });
  __syncthreads();
}

// ---- host -----------------------------------------------------------------

// A new tensor straight from the allocator: a small call's five or so take
// as long as its launches, and the way through the dispatcher is half of it.
static torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type,
                           const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
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
  // (1,024 rows at a time are addressed in 32 bits)
  TORCH_CHECK(s.hw < (1L << 31) && c < (1L << 19), "group_norm: a sample of ",
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

struct Cut {
  Slab d;
  int threads, vectors;
};

// the narrowest slice, in columns, that has whole groups and whole vectors
static int least_slice(const Shape& s, int v) {
  int a = s.cpg, b = v;
  while (b) {
    const int t = a % b;
    a = b;
    b = t;
  }
  return s.cpg / a;
}

// Threads to hold `rows` rows of the slice, and vectors for each of them. w:
// entries of a group in a row of a table, a vector's parts or its channels.
static void man(Cut& out, long rows, int top, int w) {
  Slab& d = out.d;
  const long want = ((long)d.lanes * rows + 63) / 64 * 64;
  out.threads = (int)std::min<long>(top, std::max<long>(64, want));
  d.rows = out.threads / d.lanes;
  const long need = (rows + d.rows - 1) / d.rows;
  out.vectors = 1;
  while (out.vectors < need) out.vectors *= 2;
  d.per = 1;
  d.shift = 0;
  while (d.per < 64 && 2 * d.per * d.in_slice <= out.threads) {
    d.per *= 2;
    ++d.shift;
  }
  d.w = w;
  d.down = d.per / w;
  d.right = d.per % w;
  d.by_w = div_by(w);
  d.by_lanes = div_by(d.lanes);
  d.by_rows = div_by(d.rows);
  d.by_slices = div_by(d.slices);
  d.by_chunks = div_by(d.chunks);
  d.by_subs = div_by(d.subs);
  d.by_cpg = div_by(d.cpg);
  d.inv = 1.0 / ((double)d.hw * d.cpg);
  int left = d.rows;
  for (auto& l : d.level) {
    l.to = (left + 7) / 8;
    l.n = l.to * d.lanes;
    l.step = std::max(1, out.threads / l.n);
    l.by_n = div_by(l.n);
    left = l.to;
  }
}

static void fill(Cut& out, const Shape& s, int v, int lanes, int slices) {
  Slab& d = out.d;
  d.hw = (int)s.hw;
  d.c = s.c;
  d.lanes = lanes;
  d.slices = d.subs = slices;
  d.span = s.c / v;
  d.chunks = 1;
  d.per_chunk = d.hw;
  d.groups = s.groups;
  d.cpg = s.cpg;
  d.in_slice = std::max(1, lanes * v / s.cpg);
}

// Slabs of whole samples of at most `most` vectors a thread, `threads` at
// most in a block; threads is 0 where even the narrowest slice is more.
// `channels`: groups are added up from channels, and not from vectors' parts.
static Cut cut(const Shape& s, int v, int size, int threads, int most,
               bool channels) {
  Cut out{};
  const int base = least_slice(s, v), units = s.c / v / base;
  auto fits = [&](int k) {
    const long lanes = (long)base * k;
    return lanes <= SPAN && lanes * v <= (long)SPAN * s.cpg &&
           (s.hw + SPAN / lanes - 1) / (SPAN / lanes) <= most;
  };
  if (!fits(1)) return out;
  // Wider while a row of the slice is under half a cache line, or while a
  // block has under 1,024 vectors and there are blocks to spare (two a CU).
  int best = 1;
  for (int k = 2; k <= units && fits(k); ++k) {
    if (units % k) continue;
    const bool narrow = (long)base * best * v * size < 64;
    const bool small = (long)base * best * s.hw < 1024 &&
                       s.n * (units / k) >= 512;
    if (!narrow && !small) break;
    best = k;
  }
  fill(out, s, v, base * best, units / best);
  // more threads, each with less, where there are not two blocks a CU
  const int w = channels || s.cpg % v ? s.cpg : s.cpg / v;
  if (s.n * out.d.slices < 512) man(out, s.hw, threads, w);
  if (!out.threads || (out.threads > SPAN && out.vectors > WIDE_VECTORS))
    man(out, s.hw, SPAN, w);
  return out;
}

// Chunks of rows, of CHUNK_ROWS a thread and fewer where that leaves under
// 1,024 blocks, but 4 at least. `whole`: slices have whole groups, or lie
// in one; v is narrowed where neither is possible.
static Cut chop(const Shape& s, int& v, bool whole) {
  Cut out{};
  if (!whole) {
    const int cols = s.c / v;
    const int lanes = std::min(cols, 64);
    fill(out, s, v, lanes, (cols + lanes - 1) / lanes);
  } else {
    int base = least_slice(s, v);
    if (base > BLOCK && s.cpg % v) base = least_slice(s, v = 1);
    if (base > BLOCK) {
      // a slice of one group
      const int lanes = 128;
      const int subs = (base + lanes - 1) / lanes;
      fill(out, s, v, lanes, s.groups * subs);
      out.d.subs = subs;
      out.d.span = base;
    } else {
      const int units = s.c / v / base;
      int best = 1;
      for (int k = 2; k <= units; ++k)
        if (units % k == 0 && base * k <= 64 &&
            (long)base * k * v <= (long)BLOCK * s.cpg)
          best = k;
      fill(out, s, v, base * best, units / best);
    }
  }
  Slab& d = out.d;
  const int rows = BLOCK / d.lanes;
  int most = CHUNK_ROWS;
  while (most > 4 &&
         s.n * d.slices * ((s.hw + rows * most - 1) / (rows * most)) < 1024)
    most /= 2;
  d.per_chunk = (int)std::min<long>(s.hw, (long)rows * most);
  d.chunks = (int)((s.hw + d.per_chunk - 1) / d.per_chunk);
  // (a slice of one group is all entries; sums of channels are not added up)
  const bool one = d.span * v == s.cpg;
  man(out, d.per_chunk, BLOCK,
      !whole ? 1 : one ? d.lanes : s.cpg % v ? s.cpg : s.cpg / v);
  return out;
}

}  // namespace gn
}  // namespace eg
