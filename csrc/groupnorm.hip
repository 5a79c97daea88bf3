#include "groupnorm.h"

namespace eg {
namespace gn {

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
//   M2 = sum (M2_i + count_i mean_i^2) - M mean^2,
// which in 64 bits leaves 16 digits less those of (mean / spread)^2.
// Mean and rstd are kept in 64 bits: the sign of z decides a ReLU's gradient,
// and where z is next to zero it is computed again from them.
__global__ void __launch_bounds__(JOIN) join_kernel(
    const float2* __restrict__ part, double2* __restrict__ stats, long groups,
    int per_sample, int cpg, Deal d, double eps) {
  __shared__ double slot[JOIN / 64];
  const int entries = d.chunks * cpg;
  const int down = JOIN / cpg, right = JOIN % cpg;
  const double m = (double)d.hw * cpg;
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const float2* p = part + g / per_sample * d.chunks * d.c +
                      g % per_sample * cpg;
    double s = 0, q = 0;
    int chunk = threadIdx.x / cpg, ch = threadIdx.x % cpg;
#pragma unroll 4
    for (int i = threadIdx.x; i < entries; i += JOIN) {
      const float2 e = p[(long)chunk * d.c + ch];
      const double rows = min(d.per_chunk, d.hw - chunk * d.per_chunk);
      s += rows * e.x;
      q += (double)e.y + rows * e.x * e.x;
      chunk += down;
      ch += right;
      if (ch >= cpg) {
        ch -= cpg;
        ++chunk;
      }
    }
    const double mean = add_block(s, slot) / m;
    const double var = add_block(q, slot) / m - mean * mean;
    if (threadIdx.x == 0) {
      // a variance cannot be below zero, and NaN stays NaN
      stats[g] = make_double2(mean, 1.0 / sqrt((var < 0 ? 0 : var) + eps));
    }
  }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(BLOCK) apply_kernel(
    const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
    unsigned char* __restrict__ mask, const double2* __restrict__ stats,
    const float* __restrict__ gamma, const float* __restrict__ beta,
    int groups, int cpg, Deal d) {
  const Place at(d);
  if (!at.on) return;
  const int c0 = at.col * V;
  const double2* sample = stats + (long)at.n * groups;
  float mean[V], scale[V], shift[V], limit = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const double2 st = sample[(c0 + j) / cpg];
    mean[j] = (float)st.x;
    scale[j] = (float)(gamma[c0 + j] * st.y);
    shift[j] = beta[c0 + j];
    limit = fmaxf(limit, fabsf(scale[j] * mean[j]) + 2.f * fabsf(shift[j]));
  }
  limit *= 0x1p-20f;
  const long base = ((long)at.n * d.hw + at.begin) * d.c + c0;
#pragma unroll 2
  for (int k = at.r; k < at.count; k += d.rows) {
    const long i = base + (long)k * d.c;
    Vec<T, V> a = load<T, V>(x + i), b;
    if (res) b = load<T, V>(res + i);
    auto exact = [&](int j) {
      const double2 st = sample[(c0 + j) / cpg];
      const double z = ((double)(float)x[i + j] - st.x) * st.y *
                           (double)gamma[c0 + j] + (double)beta[c0 + j];
      return res ? z + (double)(float)res[i + j] : z;
    };
    const unsigned bits = activate<T, V, V, ACT>(a, b, res, mean, scale,
                                                 shift, limit, exact);
    store<T, V>(y + i, a);
    if (ACT == RELU_BITS) mask[i / V] = (unsigned char)bits;
  }
}

// The slab in one pass. P: statistics that a thread needs, 1 where a vector
// lies within a group, else one a channel.
template <typename T, int V, int I, int P, int ACT>
__global__ void __launch_bounds__(SLAB) slab_kernel(
    const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
    unsigned char* __restrict__ mask, double2* __restrict__ stats,
    const float* __restrict__ gamma, const float* __restrict__ beta,
    double eps, Slab d) {
  __shared__ float table[SLAB * P];
  __shared__ double mean_of[SLAB];
  __shared__ double rstd_of[SLAB];
  const Spot at(d, V);
  const int w = P == 1 ? d.cpg / V : d.cpg;
  const double m = (double)d.hw * d.cpg;
  const long base = (long)at.n * d.hw * d.c + at.first + at.lane * V;
  Vec<T, V> a[I];
#pragma unroll
  for (int k = 0; k < I; ++k) {
    const int row = at.r + k * d.rows;
    if (at.on && row < d.hw) a[k] = load<T, V>(x + base + (long)row * d.c);
  }
  float s[P] = {};
#pragma unroll
  for (int k = 0; k < I; ++k) {
    if (at.on && at.r + k * d.rows < d.hw) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[P == 1 ? 0 : j] += (float)a[k].v[j];
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j) table[threadIdx.x * P + j] = s[j];
  __syncthreads();
  add_groups<double>(table, d.rows, w, d,
                     [&](int q, double t) { mean_of[q] = t / m; });
  __syncthreads();
  float mean[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    mean[j] = (float)mean_of[(at.lane * V + j) / d.cpg];
    s[j] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < I; ++k) {
    if (at.on && at.r + k * d.rows < d.hw) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int p = P == 1 ? 0 : j;
        const float e = (float)a[k].v[j] - mean[p];
        s[p] = fmaf(e, e, s[p]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j) table[threadIdx.x * P + j] = s[j];
  __syncthreads();
  add_groups<double>(table, d.rows, w, d, [&](int q, double t) {
    const double rstd = 1.0 / sqrt(t / m + eps);
    rstd_of[q] = rstd;
    if (stats)
      stats[(long)at.n * d.groups + at.first / d.cpg + q] =
          make_double2(mean_of[q], rstd);
  });
  __syncthreads();
  if (!at.on) return;
  const int c0 = at.first + at.lane * V;
  float scale[V], shift[V], limit = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int p = P == 1 ? 0 : j;
    scale[j] = (float)(gamma[c0 + j] * rstd_of[(at.lane * V + p) / d.cpg]);
    shift[j] = beta[c0 + j];
    limit = fmaxf(limit, fabsf(scale[j] * mean[p]) + 2.f * fabsf(shift[j]));
  }
  limit *= 0x1p-20f;
#pragma unroll
  for (int k = 0; k < I; ++k) {
    const int row = at.r + k * d.rows;
    if (row >= d.hw) break;
    const long i = base + (long)row * d.c;
    Vec<T, V> b;
    if (res) b = load<T, V>(res + i);
    auto exact = [&](int j) {
      const int q = (at.lane * V + j) / d.cpg;
      const double z = ((double)(float)x[i + j] - mean_of[q]) * rstd_of[q] *
                           (double)gamma[c0 + j] + (double)beta[c0 + j];
      return res ? z + (double)(float)res[i + j] : z;
    };
    const unsigned bits = activate<T, V, P, ACT>(a[k], b, res, mean, scale,
                                                 shift, limit, exact);
    store<T, V>(y + i, a[k]);
    if (ACT == RELU_BITS) mask[i / V] = (unsigned char)bits;
  }
}

}  // namespace gn

// y; and where `stats` is given per sample and group (mean, rstd) in 64 bits,
// and for a ReLU the bits of z > 0
static torch::Tensor forward(const torch::Tensor& x,
                             const torch::Tensor& gamma,
                             const torch::Tensor& beta, const gn::Shape& s,
                             double eps, long act, const torch::Tensor& res,
                             torch::Tensor* stats, torch::Tensor* mask) {
  using namespace gn;
  TORCH_CHECK(eps >= 0, "group_norm: eps must not be negative");
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty_like(x);
  const auto f64 = x.options().dtype(torch::kFloat64);
  if (stats) *stats = torch::empty({s.n, s.groups, 2}, f64);
  if (x.numel() == 0) return y;
  const void* r = res.defined() ? res.data_ptr() : nullptr;
  const int size = (int)x.element_size();
  const int v = width(s, size, {x.data_ptr(), y.data_ptr(), r});
  const float* gm = gamma.data_ptr<float>();
  const float* bt = beta.data_ptr<float>();
  unsigned char* mk = nullptr;
  if (mask && act == RELU) {
    *mask = torch::empty({x.numel() / v}, x.options().dtype(torch::kUInt8));
    mk = mask->data_ptr<unsigned char>();
  }
  const hipStream_t stream = cur_stream();
  const Cut slab = cut(s, v, size, FWD_VECTORS);
  if (slab.threads) {
    auto* st = stats ? reinterpret_cast<double2*>(stats->data_ptr()) : nullptr;
    with_slab(x.scalar_type(), v, slab.vectors, s.cpg % v == 0, [&](auto tag) {
      using G = decltype(tag);
      using T = typename G::type;
      if constexpr (G::i <= FWD_VECTORS) {
        with_act(act, mk, [&](auto a) {
          slab_kernel<T, G::v, G::i, G::p, decltype(a)::v>
              <<<(unsigned)(s.n * slab.d.slices), slab.threads, 0, stream>>>(
                  reinterpret_cast<const T*>(x.data_ptr()),
                  reinterpret_cast<const T*>(r),
                  reinterpret_cast<T*>(y.data_ptr()), mk, st, gm, bt, eps,
                  slab.d);
        });
      }
    });
    return y;
  }
  torch::Tensor own = stats ? *stats : torch::empty({s.n, s.groups, 2}, f64);
  const Deal d = deal(s.hw, s.c, v, s.n);
  auto part = torch::empty({s.n, d.chunks, s.c, 2},
                           x.options().dtype(torch::kFloat32));
  const dim3 grid((unsigned)(s.n * d.chunks), 1,
                  (unsigned)((d.cols + d.lanes - 1) / d.lanes));
  const long all = s.n * s.groups;
  const unsigned joins = (unsigned)std::min<long>(all, 1 << 20);
  auto* st = reinterpret_cast<double2*>(own.data_ptr());
  auto* pt = reinterpret_cast<float2*>(part.data_ptr());
  with_type(x.scalar_type(), v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    const T* xp = reinterpret_cast<const T*>(x.data_ptr());
    stats_kernel<T, V><<<grid, BLOCK, 0, stream>>>(xp, pt, d);
    join_kernel<<<joins, JOIN, 0, stream>>>(pt, st, all, s.groups, s.cpg, d,
                                             eps);
    with_act(act, mk, [&](auto a) {
      apply_kernel<T, V, decltype(a)::v><<<grid, BLOCK, 0, stream>>>(
          xp, reinterpret_cast<const T*>(r),
          reinterpret_cast<T*>(y.data_ptr()), mk, st, gm, bt, s.groups, s.cpg,
          d);
    });
  });
  return y;
}

// y, and the statistics and bits that group_norm_bwd takes
std::vector<torch::Tensor> group_norm_fwd(torch::Tensor x,
                                          torch::Tensor gamma,
                                          torch::Tensor beta, long groups,
                                          double eps, long act,
                                          c10::optional<torch::Tensor> res) {
  const auto s = gn::shape_of(x, gamma, beta, groups, act, res);
  torch::Tensor stats, mask;
  auto y = forward(x, gamma, beta, s, eps, act,
                   res ? *res : torch::Tensor(), &stats, &mask);
  return {y, stats, mask};
}

// y alone
torch::Tensor group_norm_only(torch::Tensor x, torch::Tensor gamma,
                              torch::Tensor beta, long groups, double eps,
                              long act, c10::optional<torch::Tensor> res) {
  const auto s = gn::shape_of(x, gamma, beta, groups, act, res);
  return forward(x, gamma, beta, s, eps, act, res ? *res : torch::Tensor(),
                 nullptr, nullptr);
}

}  // namespace eg
