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
// Nothing here adds in an order that changes: every sum goes through slots
// of its own that are added in a fixed order.

#include "common.h"

#include <c10/core/DeviceGuard.h>

namespace eg {
namespace gn {

constexpr int BLOCK = 256;
enum Act { NONE = 0, RELU = 1, SILU = 2 };

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

__device__ __forceinline__ float sigmoid(float z) {
  return 1.f / (1.f + __expf(-z));
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == RELU) return z < 0.f ? 0.f : z;   // NaN stays NaN
  if (act == SILU) return z * sigmoid(z);
  return z;
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

// ---- forward --------------------------------------------------------------

// Each channel's mean and sum of squared distances from it over one chunk of
// rows. Distances are first measured from the chunk's own first value, which
// is among those it adds, so that a large mean costs no digits.
template <typename T, int V>
__global__ void __launch_bounds__(BLOCK) stats_kernel(
    const T* __restrict__ x, float2* __restrict__ part, Deal d) {
  __shared__ float slot[BLOCK / 2 * 2 * V];
  const Place at(d);
  float from[V] = {}, sums[2 * V] = {};
  if (at.on) {
    const T* xs = x + ((long)at.n * d.hw + at.begin) * d.c + at.col * V;
    const Vec<T, V> f = load<T, V>(xs);
#pragma unroll
    for (int j = 0; j < V; ++j) from[j] = (float)f.v[j];
#pragma unroll 4
    for (int k = at.r; k < at.count; k += d.rows) {
      const Vec<T, V> a = load<T, V>(xs + (long)k * d.c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float e = (float)a.v[j] - from[j];
        sums[j] += e;
        sums[V + j] = fmaf(e, e, sums[V + j]);
      }
    }
  }
  add_rows<2 * V>(sums, slot, at.r, at.lane, d.lanes, d.rows);
  if (at.on && at.r == 0) {
    float2* to = part + (long)blockIdx.x * d.c + at.col * V;
    const float inv = 1.f / (float)at.count;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float off = sums[j] * inv;
      to[j] = make_float2(from[j] + off, fmaf(-sums[j], off, sums[V + j]));
    }
  }
}

// One block a group: joins the channels and chunks of each,
//   M2 = sum M2_i + count_i (mean_i - mean)^2.
// Mean and rstd are kept in 64 bits: the sign of z decides a ReLU's gradient,
// and where z is next to zero it is computed again from them.
__global__ void __launch_bounds__(BLOCK) join_kernel(
    const float2* __restrict__ part, double2* __restrict__ stats, long groups,
    int per_sample, int cpg, Deal d, double eps) {
  __shared__ double slot[BLOCK / 64];
  const long entries = (long)d.chunks * cpg;
  const double m = (double)d.hw * cpg;
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const float2* p = part + g / per_sample * d.chunks * d.c +
                      g % per_sample * cpg;
    double s = 0;
    for (long i = threadIdx.x; i < entries; i += BLOCK) {
      const int chunk = (int)(i / cpg);
      const int rows = min(d.per_chunk, d.hw - chunk * d.per_chunk);
      s += (double)rows * p[(long)chunk * d.c + i % cpg].x;
    }
    const double mean = add_block(s, slot) / m;
    double q = 0;
    for (long i = threadIdx.x; i < entries; i += BLOCK) {
      const int chunk = (int)(i / cpg);
      const int rows = min(d.per_chunk, d.hw - chunk * d.per_chunk);
      const float2 e = p[(long)chunk * d.c + i % cpg];
      const double off = (double)e.x - mean;
      q += (double)e.y + (double)rows * off * off;
    }
    const double var = add_block(q, slot) / m;
    if (threadIdx.x == 0) {
      // a variance cannot be below zero, and NaN stays NaN
      stats[g] = make_double2(mean, 1.0 / sqrt((var < 0 ? 0 : var) + eps));
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(BLOCK) apply_kernel(
    const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
    const double2* __restrict__ stats, const float* __restrict__ gamma,
    const float* __restrict__ beta, int groups, int cpg, int act, Deal d) {
  const Place at(d);
  if (!at.on) return;
  float mean[V], scale[V], shift[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int ch = at.col * V + j;
    const double2 st = stats[(long)at.n * groups + ch / cpg];
    mean[j] = (float)st.x;
    scale[j] = (float)(gamma[ch] * st.y);
    shift[j] = beta[ch];
  }
  const long base = ((long)at.n * d.hw + at.begin) * d.c + at.col * V;
#pragma unroll 2
  for (int k = at.r; k < at.count; k += d.rows) {
    const long i = base + (long)k * d.c;
    Vec<T, V> a = load<T, V>(x + i), b;
    if (res) b = load<T, V>(res + i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float z = fmaf((float)a.v[j] - mean[j], scale[j], shift[j]);
      if (res) z += (float)b.v[j];
      a.v[j] = (T)activate(z, act);
    }
    store<T, V>(y + i, a);
  }
}

// ---- backward -------------------------------------------------------------

// What a thread keeps of its V channels, and dz from them.
template <typename T, int V>
struct Channels {
  float mean[V], rstd[V], gamma[V], beta[V];
  const double2* stats;
  int cpg, first;

  __device__ __forceinline__ Channels(const double2* sample, int c0,
                                      const float* g, const float* b, int n) {
    stats = sample;
    cpg = n;
    first = c0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double2 st = sample[(c0 + j) / n];
      mean[j] = (float)st.x;
      rstd[j] = (float)st.y;
      gamma[j] = g[c0 + j];
      beta[j] = b[c0 + j];
    }
  }

  // xh, and dz = dy act'(z). z is off by a few 2^-24 of the terms that make
  // it; where that could turn its sign it is taken again in 64 bits.
  __device__ __forceinline__ float dz(int j, float x, float r, float dy,
                                      int act, float& xh) const {
    xh = (x - mean[j]) * rstd[j];
    if (act == NONE) return dy;
    float z = fmaf(xh, gamma[j], beta[j]) + r;
    if (act == SILU) {
      const float s = sigmoid(z);
      return dy * (s * fmaf(z, 1.f - s, 1.f));
    }
    const float unsure =
        0x1p-20f * (fabsf(gamma[j] * rstd[j] * mean[j]) +
                    2.f * (fabsf(beta[j]) + fabsf(r)));
    if (fabsf(z) <= unsure) {
      const double2 st = stats[(first + j) / cpg];
      const double e = ((double)x - st.x) * st.y * (double)gamma[j] +
                       (double)beta[j] + (double)r;
      return e <= 0.0 ? 0.f : dy;
    }
    return z <= 0.f ? 0.f : dy;
  }
};

// Each channel's sums of dz and of dz xh over one chunk of rows.
template <typename T, int V>
__global__ void __launch_bounds__(BLOCK) bwd_sums_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const double2* __restrict__ stats,
    const float* __restrict__ gamma, const float* __restrict__ beta,
    float2* __restrict__ part, int groups, int cpg, int act, Deal d) {
  __shared__ float slot[BLOCK / 2 * 2 * V];
  const Place at(d);
  float sums[2 * V] = {};
  if (at.on) {
    const Channels<T, V> ch(stats + (long)at.n * groups, at.col * V, gamma,
                            beta, cpg);
    const long base = ((long)at.n * d.hw + at.begin) * d.c + at.col * V;
#pragma unroll 2
    for (int k = at.r; k < at.count; k += d.rows) {
      const long i = base + (long)k * d.c;
      const Vec<T, V> a = load<T, V>(x + i), g = load<T, V>(dy + i);
      Vec<T, V> b;
      if (res) b = load<T, V>(res + i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float xh;
        const float dz = ch.dz(j, (float)a.v[j], res ? (float)b.v[j] : 0.f,
                               (float)g.v[j], act, xh);
        sums[j] += dz;
        sums[V + j] = fmaf(dz, xh, sums[V + j]);
      }
    }
  }
  add_rows<2 * V>(sums, slot, at.r, at.lane, d.lanes, d.rows);
  if (at.on && at.r == 0) {
    float2* to = part + (long)blockIdx.x * d.c + at.col * V;
#pragma unroll
    for (int j = 0; j < V; ++j) to[j] = make_float2(sums[j], sums[V + j]);
  }
}

// One block a group: each channel's sums over the chunks, for dgamma and
// dbeta, and the group's s1 and s2.
__global__ void __launch_bounds__(BLOCK) bwd_join_kernel(
    const float2* __restrict__ part, const float* __restrict__ gamma,
    float2* __restrict__ channel, float2* __restrict__ group, long groups,
    int per_sample, int cpg, int across, Deal d) {
  // across: threads side by side over channels, a power of two
  __shared__ float2 slot[BLOCK];
  __shared__ float sums[BLOCK / 64];
  const int lane = threadIdx.x % across, share = threadIdx.x / across;
  const int shares = BLOCK / across;
  const float inv = 1.f / ((float)d.hw * (float)cpg);
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const long n = g / per_sample;
    const int c0 = (int)(g % per_sample) * cpg;
    float s1 = 0.f, s2 = 0.f;
    for (int b = 0; b < cpg; b += across) {
      const bool on = b + lane < cpg;
      float2 s = make_float2(0.f, 0.f);
      if (on) {
        const float2* p = part + n * d.chunks * d.c + c0 + b + lane;
        for (int k = share; k < d.chunks; k += shares) {
          const float2 e = p[(long)k * d.c];
          s.x += e.x;
          s.y += e.y;
        }
      }
      for (int half = shares / 2; half; half /= 2) {
        if (share >= half && share < 2 * half)
          slot[threadIdx.x - half * across] = s;
        __syncthreads();
        if (share < half) {
          s.x += slot[threadIdx.x].x;
          s.y += slot[threadIdx.x].y;
        }
        __syncthreads();
      }
      if (on && share == 0) {
        channel[n * d.c + c0 + b + lane] = s;
        s1 = fmaf(gamma[c0 + b + lane], s.x, s1);
        s2 = fmaf(gamma[c0 + b + lane], s.y, s2);
      }
    }
    s1 = add_block(s1, sums);
    s2 = add_block(s2, sums);
    if (threadIdx.x == 0) group[g] = make_float2(s1 * inv, s2 * inv);
  }
}

// dgamma and dbeta: each channel's sums over the samples, added to what is
// there (a gradient's view in the flat space) or put down.
constexpr int PC = 32, PN = 32;
__global__ void __launch_bounds__(PC* PN) bwd_params_kernel(
    const float2* __restrict__ channel, float* __restrict__ dgamma,
    float* __restrict__ dbeta, long n, int c, int add) {
  __shared__ float2 slot[PN / 2][PC];
  const int lane = threadIdx.x % PC, share = threadIdx.x / PC;
  const int ch = blockIdx.x * PC + lane;
  float2 s = make_float2(0.f, 0.f);
  if (ch < c) {
    for (long k = share; k < n; k += PN) {
      const float2 e = channel[k * c + ch];
      s.x += e.x;
      s.y += e.y;
    }
  }
  for (int half = PN / 2; half; half /= 2) {
    if (share >= half && share < 2 * half) slot[share - half][lane] = s;
    __syncthreads();
    if (share < half) {
      s.x += slot[share][lane].x;
      s.y += slot[share][lane].y;
    }
    __syncthreads();
  }
  if (share == 0 && ch < c) {
    dgamma[ch] = add ? dgamma[ch] + s.y : s.y;
    dbeta[ch] = add ? dbeta[ch] + s.x : s.x;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(BLOCK) bwd_apply_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const double2* __restrict__ stats,
    const float* __restrict__ gamma, const float* __restrict__ beta,
    const float2* __restrict__ group, T* __restrict__ dx,
    T* __restrict__ dres, int groups, int cpg, int act, Deal d) {
  const Place at(d);
  if (!at.on) return;
  const Channels<T, V> ch(stats + (long)at.n * groups, at.col * V, gamma,
                          beta, cpg);
  float s1[V], s2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float2 s = group[(long)at.n * groups + (at.col * V + j) / cpg];
    s1[j] = s.x;
    s2[j] = s.y;
  }
  const long base = ((long)at.n * d.hw + at.begin) * d.c + at.col * V;
#pragma unroll 2
  for (int k = at.r; k < at.count; k += d.rows) {
    const long i = base + (long)k * d.c;
    const Vec<T, V> a = load<T, V>(x + i), g = load<T, V>(dy + i);
    Vec<T, V> b, u;
    if (res) b = load<T, V>(res + i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float xh;
      const float dz = ch.dz(j, (float)a.v[j], res ? (float)b.v[j] : 0.f,
                             (float)g.v[j], act, xh);
      u.v[j] = (T)(ch.rstd[j] *
                   (fmaf(dz, ch.gamma[j], -s1[j]) - xh * s2[j]));
      b.v[j] = (T)dz;
    }
    if (dx) store<T, V>(dx + i, u);
    if (dres) store<T, V>(dres + i, b);
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
  // about 2,048 blocks, eight a CU, and no chunk under four rows a thread
  const long wanted = std::max<long>(1, 2048 / std::max<long>(1, n * tiles));
  const long most = std::max<long>(1, hw / (4L * d.rows));
  const long chunks = std::min(wanted, most);
  d.per_chunk = (int)((hw + chunks - 1) / chunks);
  d.chunks = (int)((hw + d.per_chunk - 1) / d.per_chunk);
  return d;
}

struct Shape {
  long n, hw, blocks;
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

}  // namespace gn

// y and, per sample and group, (mean, rstd) in 64 bits
std::vector<torch::Tensor> group_norm_fwd(torch::Tensor x,
                                          torch::Tensor gamma,
                                          torch::Tensor beta, long groups,
                                          double eps, long act,
                                          c10::optional<torch::Tensor> res) {
  using namespace gn;
  const Shape s = shape_of(x, gamma, beta, groups, act, res);
  TORCH_CHECK(eps >= 0, "group_norm: eps must not be negative");
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty_like(x);
  auto stats = torch::empty({s.n, groups, 2}, x.options().dtype(torch::kFloat64));
  if (x.numel() == 0) return {y, stats};
  const void* r = res ? res->data_ptr() : nullptr;
  const int v = width(s, (int)x.element_size(),
                      {x.data_ptr(), y.data_ptr(), r});
  const Deal d = deal(s.hw, s.c, v, s.n);
  auto part = torch::empty({s.n, d.chunks, s.c, 2},
                           x.options().dtype(torch::kFloat32));
  const dim3 grid((unsigned)(s.n * d.chunks), 1,
                  (unsigned)((d.cols + d.lanes - 1) / d.lanes));
  const long all = s.n * groups;
  const unsigned joins = (unsigned)std::min<long>(all, 1 << 20);
  auto* st = reinterpret_cast<double2*>(stats.data_ptr());
  auto* pt = reinterpret_cast<float2*>(part.data_ptr());
  with_type(x.scalar_type(), v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    const T* xp = reinterpret_cast<const T*>(x.data_ptr());
    stats_kernel<T, V><<<grid, BLOCK, 0, cur_stream()>>>(xp, pt, d);
    join_kernel<<<joins, BLOCK, 0, cur_stream()>>>(pt, st, all, s.groups,
                                                   s.cpg, d, eps);
    apply_kernel<T, V><<<grid, BLOCK, 0, cur_stream()>>>(
        xp, reinterpret_cast<const T*>(r),
        reinterpret_cast<T*>(y.data_ptr()), st, gamma.data_ptr<float>(),
        beta.data_ptr<float>(), s.groups, s.cpg, (int)act, d);
  });
  return {y, stats};
}

// dx, the residual's gradient, dgamma and dbeta; an undefined tensor where
// one is not wanted. The parameters' gradients are added to dgamma_out and
// dbeta_out where those are given.
std::vector<torch::Tensor> group_norm_bwd(
    torch::Tensor dy, torch::Tensor x, torch::Tensor stats,
    torch::Tensor gamma, torch::Tensor beta, long groups, long act,
    c10::optional<torch::Tensor> res, bool want_dx, bool want_dres,
    c10::optional<torch::Tensor> dgamma_out,
    c10::optional<torch::Tensor> dbeta_out) {
  using namespace gn;
  const Shape s = shape_of(x, gamma, beta, groups, act, res);
  TORCH_CHECK(dy.device() == x.device() &&
                  dy.scalar_type() == x.scalar_type() &&
                  dy.sizes() == x.sizes() && dy.is_contiguous(),
              "group_norm: dy must be like x, and contiguous");
  TORCH_CHECK(stats.device() == x.device() &&
                  stats.scalar_type() == torch::kFloat64 &&
                  stats.is_contiguous() && stats.numel() == 2 * s.n * groups,
              "group_norm: stats must be those of the forward pass");
  const bool add = dgamma_out.has_value();
  TORCH_CHECK(add == dbeta_out.has_value(),
              "group_norm: dgamma_out and dbeta_out go together");
  const c10::DeviceGuard guard(x.device());
  const auto f32 = x.options().dtype(torch::kFloat32);
  torch::Tensor dx, dres, dgamma, dbeta;
  if (want_dx) dx = torch::empty_like(x);
  if (want_dres) dres = torch::empty_like(x);
  if (add) {
    dgamma = *dgamma_out;
    dbeta = *dbeta_out;
    for (const auto& t : {dgamma, dbeta})
      TORCH_CHECK(t.device() == x.device() &&
                      t.scalar_type() == torch::kFloat32 &&
                      t.is_contiguous() && t.numel() == s.c,
                  "group_norm: gradient views must be contiguous fp32 "
                  "vectors of ", s.c);
  } else {
    dgamma = torch::empty({s.c}, f32);
    dbeta = torch::empty({s.c}, f32);
  }
  if (x.numel() == 0) {
    if (!add) {
      dgamma.zero_();
      dbeta.zero_();
    }
    return {dx, dres, dgamma, dbeta};
  }
  const void* r = res ? res->data_ptr() : nullptr;
  void* dxp = want_dx ? dx.data_ptr() : nullptr;
  void* drp = want_dres ? dres.data_ptr() : nullptr;
  const int v = width(s, (int)x.element_size(),
                      {x.data_ptr(), dy.data_ptr(), r, dxp, drp});
  const Deal d = deal(s.hw, s.c, v, s.n);
  auto part = torch::empty({s.n, d.chunks, s.c, 2}, f32);
  auto channel = torch::empty({s.n, s.c, 2}, f32);
  auto group = torch::empty({s.n, groups, 2}, f32);
  const dim3 grid((unsigned)(s.n * d.chunks), 1,
                  (unsigned)((d.cols + d.lanes - 1) / d.lanes));
  const long all = s.n * groups;
  const unsigned joins = (unsigned)std::min<long>(all, 1 << 20);
  const auto* st = reinterpret_cast<const double2*>(stats.data_ptr());
  auto* pt = reinterpret_cast<float2*>(part.data_ptr());
  auto* cp = reinterpret_cast<float2*>(channel.data_ptr());
  auto* gp = reinterpret_cast<float2*>(group.data_ptr());
  const float* gm = gamma.data_ptr<float>();
  const float* bt = beta.data_ptr<float>();
  int across = 1;
  while (across < s.cpg && across < BLOCK) across *= 2;
  with_type(x.scalar_type(), v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    const T* xp = reinterpret_cast<const T*>(x.data_ptr());
    const T* yp = reinterpret_cast<const T*>(dy.data_ptr());
    const T* rp = reinterpret_cast<const T*>(r);
    bwd_sums_kernel<T, V><<<grid, BLOCK, 0, cur_stream()>>>(
        yp, xp, rp, st, gm, bt, pt, s.groups, s.cpg, (int)act, d);
    bwd_join_kernel<<<joins, BLOCK, 0, cur_stream()>>>(
        pt, gm, cp, gp, all, s.groups, s.cpg, across, d);
    bwd_params_kernel<<<ceil_div(s.c, PC), PC * PN, 0, cur_stream()>>>(
        cp, dgamma.data_ptr<float>(), dbeta.data_ptr<float>(), s.n, s.c,
        add ? 1 : 0);
    if (dxp || drp)
      bwd_apply_kernel<T, V><<<grid, BLOCK, 0, cur_stream()>>>(
          yp, xp, rp, st, gm, bt, gp, reinterpret_cast<T*>(dxp),
          reinterpret_cast<T*>(drp), s.groups, s.cpg, (int)act, d);
  });
  return {dx, dres, dgamma, dbeta};
}

}  // namespace eg
