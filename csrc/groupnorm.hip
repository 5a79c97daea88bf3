#include "groupnorm.h"

namespace eg {
namespace gn {

// rows that a thread has in flight: on 1x512x512x128 the statistics took 14.6 us
// with 4 and 15.0 with 8 (14.4 with both on 4x128x128x320), applying them 22.3
// with 4 and 22.7 with 2 (16.3 and 16.6)
constexpr int STATS_AT_ONCE = 4, APPLY_AT_ONCE = 4;

// values of a group in `rows` rows of a slab: the group's, or where a slice
// is one of several in a group those of slice `sub`
__device__ __forceinline__ double piece(const Slab& d, int v, int rows,
                                        int sub) {
  const int wide = d.span * v == d.cpg
                       ? min(d.lanes, d.span - sub * d.lanes) * v
                       : d.cpg;
  return (double)rows * wide;
}

// ---- forward --------------------------------------------------------------

// Each group's mean and sum of squared distances from it over one chunk of
// rows; about 1,024 blocks, with 4 to 16 rows a thread, since the block's own
// sums cost as much as some rows. 1x512x512x128 bf16: 67 MB in 14.6 us, 4.6
// TB/s; a form that held its rows in registers and summed once for 48 of them
// took 21. Distances are first measured from the group's first value in the
// chunk, which is among those added, so that a large mean costs no digits.
// EXACT: the distances, their squares and all sums are in 64 bits, for a
// ReLU's bits hang on them (0.7 us of 41.6 on 1x512x512x128, nothing on
// 4x128x128x320). Else a vector's are in fp32, or with P > 1 a channel's in
// one thread.
template <typename T, int V, int P, bool EXACT>
__global__ void __launch_bounds__(BLOCK) stats_kernel(
    const T* __restrict__ x, double2* __restrict__ part_of, Slab d) {
  __shared__ double table[2 * BLOCK * P];
  __shared__ float from_of[BLOCK];
  const Spot at(d, V);
  // entries of a group: its slices, and the chunks of each
  const bool alone = d.span * V == d.cpg;
  const int unit = d.by_subs.of(at.slice);
  const int subs = alone ? d.subs : 1;
  const int sub = alone ? at.slice - unit * d.subs : 0;
  const int group = alone ? unit : at.slice * d.in_slice;
  const T* row0 = x + ((long)at.n * d.hw + at.begin) * d.c;
  using Sum = std::conditional_t<P == 1 || EXACT, double, float>;
  using Off = std::conditional_t<EXACT, double, float>;
  float from[P];
  Sum s[P] = {}, q2[P] = {};
  each_part<P>(alone ? 0 : at.lane * V, d, [&](int j, int q) {
    from[j] = (float)row0[(long)(group + q) * d.cpg];
  });
  each_row<STATS_AT_ONCE>(at, d, [&](int k) {
    const Vec<T, V> a = load<T, V>(at.row(x, k));
    Off t = 0, t2 = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const Off e = (Off)a[j] - from[P == 1 ? 0 : j];
      if (P == 1) {
        t += e;
        t2 = __builtin_elementwise_fma(e, e, t2);
      } else {
        s[j] += e;
        q2[j] = __builtin_elementwise_fma(e, e, (Off)q2[j]);
      }
    }
    if (P == 1) {
      s[0] += t;
      q2[0] += t2;
    }
  });
#pragma unroll
  for (int j = 0; j < P; ++j) {
    table[j * blockDim.x + threadIdx.x] = s[j];
    table[(P + j) * blockDim.x + threadIdx.x] = q2[j];
  }
  for (int q = threadIdx.x; q < d.in_slice; q += blockDim.x)
    from_of[q] = (float)row0[(long)(group + q) * d.cpg];
  __syncthreads();
  const int rows = fold<2 * P>(table, d, P == 1 ? BLOCK : 8);
  const double values = piece(d, V, at.count, sub);
  add_groups<Twice>(
      rows, d,
      [&](int e, int row) {
        return Twice{part<P>(table, d, e, row),
                     part<P>(table + P * blockDim.x, d, e, row)};
      },
      [&](int q, const Twice& t) {
        const double off = t.a / values;
        part_of[(((long)at.n * d.groups + group + q) * subs + sub) * d.chunks +
                at.chunk] =
            make_double2(from_of[q] + off, t.b - t.a * off);
      });
}

// Joins the pieces of each group, a block for each,
//   M2 = sum (M2_i + count_i off_i^2) - M off^2,
// off being measured from the first piece's mean: from zero it would cost the
// digits of (mean / spread)^2.
// Mean and rstd are kept in 64 bits: the sign of z decides a ReLU's gradient,
// and where z is next to zero it is computed again from them.
__global__ void __launch_bounds__(BLOCK) join_kernel(
    const double2* __restrict__ part, double2* __restrict__ stats, long groups,
    int v, Slab d, double eps) {
  __shared__ double slot[BLOCK / 64];
  const bool alone = d.span * v == d.cpg;
  const int subs = alone ? d.subs : 1;
  const double m = (double)d.hw * d.cpg;
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const double2* p = part + g * subs * d.chunks;
    const double from = p[0].x;
    double s = 0, q = 0;
    for (int i = threadIdx.x; i < subs * d.chunks; i += blockDim.x) {
      const int chunk = i % d.chunks;
      const double n =
          piece(d, v, min(d.per_chunk, d.hw - chunk * d.per_chunk),
                i / d.chunks);
      const double2 e = p[i];
      const double off = e.x - from;
      s += n * off;
      q += e.y + n * off * off;
    }
    const double off = add_block(s, slot) / m;
    const double var = add_block(q, slot) / m - off * off;
    if (threadIdx.x == 0) {
      // a variance cannot be below zero, and NaN stays NaN
      stats[g] = make_double2(from + off,
                              1.0 / sqrt((var < 0 ? 0 : var) + eps));
    }
  }
}

// y from the statistics: a second reading of x, which is then in the last-level
// cache up to some 200 MB. 1x512x512x128 bf16: 134 MB in 22.3 us, 6.0 TB/s.
template <typename T, int V, int P, int ACT>
__global__ void __launch_bounds__(BLOCK) apply_kernel(
    const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
    unsigned char* __restrict__ mask, const double2* __restrict__ stats,
    const float* __restrict__ gamma, const float* __restrict__ beta, Slab d) {
  const Spot at(d, V);
  const int c0 = at.first;
  const double2* sample = stats + (long)at.n * d.groups;
  float mean[P], scale[V], shift[V], limit = 0.f;
  double2 st[P];
  each_part<P>(c0, d, [&](int j, int q) { st[j] = sample[q]; });
#pragma unroll
  for (int j = 0; j < P; ++j) mean[j] = (float)st[j].x;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int p = P == 1 ? 0 : j;
    scale[j] = (float)(gamma[c0 + j] * st[p].y);
    shift[j] = fmaf(-(float)(st[p].x - mean[p]), scale[j], beta[c0 + j]);
    limit = fmaxf(limit, fabsf(scale[j] * mean[p]) + 2.f * fabsf(shift[j]));
  }
  limit *= 0x1p-20f;
  each_row<APPLY_AT_ONCE>(at, d, [&](int k) {
    Vec<T, V> a = load<T, V>(at.row(x, k)), b;
    if (res) b = load<T, V>(at.row(res, k));
    auto exact = [&](int j) {
      const double2 st = sample[d.by_cpg.of(c0 + j)];
      const double z = ((double)(float)at.row(x, k)[j] - st.x) * st.y *
                           (double)gamma[c0 + j] + (double)beta[c0 + j];
      return res ? z + (double)(float)at.row(res, k)[j] : z;
    };
    const unsigned bits = activate<T, V, P, ACT>(a, b, res, mean, scale, shift,
                                                 limit, exact);
    store<T, V>(at.row(y, k), a);
    if (ACT == RELU_BITS) *at.template bits<V>(mask, k) = (unsigned char)bits;
  });
}

// All of it in one pass over a slab of whole samples: 102 MB of
// 256x32x32x64 bf16 with residual, ReLU and bits in 27.9 us, 3.7 TB/s (26.5
// with sums in fp32, which are too rough for the bits). All blocks are on the
// chip at once: they load, add up and write in step, and the caches are
// written back behind them. Loading the residual ahead of the sums, lines of
// 128 bytes with twice the vectors and of 32 bytes were no better (28.5, 26.4
// and 32.2 us to 26.5).
template <typename T, int V, int I, int P, int ACT>
__global__ void __launch_bounds__(I <= WIDE_VECTORS ? fwd_threads(P)
                                                    : SPAN) slab_kernel(
    const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
    unsigned char* __restrict__ mask, double2* __restrict__ stats,
    const float* __restrict__ gamma, const float* __restrict__ beta,
    double eps, Slab d) {
  __shared__ double table[(I <= WIDE_VECTORS ? fwd_threads(P) : SPAN) * P];
  __shared__ double mean_of[SPAN];
  __shared__ double rstd_of[SPAN];
  __shared__ float low_of[SPAN];    // rstd times what the mean is rounded by
  const Spot at(d, V);
  Vec<T, V> a[I];
#pragma unroll
  for (int k = 0; k < I; ++k)
    if (at.has(k, d)) a[k] = load<T, V>(at.row(x, k));
  const int c0 = at.first;
  float scale[V], shift[V], mean[P];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    scale[j] = gamma[c0 + j];
    shift[j] = beta[c0 + j];
  }
  // (a ReLU gives the same values with its bits and without)
  statistics<T, V, I, P, ACT == RELU || ACT == RELU_BITS>(
      a, at, d, table, mean_of, mean, [&](int q, double mu, double m2) {
        const double rstd = 1.0 / sqrt(m2 * d.inv + eps);
        rstd_of[q] = rstd;
        low_of[q] = (float)((mu - (float)mu) * rstd);
        if (stats)
          stats[(long)at.n * d.groups + at.slice * d.in_slice + q] =
              make_double2(mu, rstd);
      });
  if (!at.on) return;
  float limit = 0.f;
  if (P == 1) {
    const int q = d.by_cpg.of(at.lane * V);
    const double rstd = rstd_of[q];
    const float low = low_of[q];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      shift[j] = fmaf(-low, scale[j], shift[j]);
      scale[j] = (float)(scale[j] * rstd);
    }
  } else {
    each_part<P>(at.lane * V, d, [&](int j, int q) {
      shift[j] = fmaf(-low_of[q], scale[j], shift[j]);
      scale[j] = (float)(scale[j] * rstd_of[q]);
    });
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    limit = fmaxf(limit, fabsf(scale[j] * mean[P == 1 ? 0 : j]) +
                             2.f * fabsf(shift[j]));
  limit *= 0x1p-20f;
#pragma unroll
  for (int k = 0; k < I; ++k) {
    if (!at.has(k, d)) break;
    renew<T, V>(a[k]);
    Vec<T, V> b;
    if (res) b = load<T, V>(at.row(res, k));
    auto exact = [&](int j) {
      const int q = (at.lane * V + j) / d.cpg;
      const double z = ((double)(float)at.row(x, k)[j] - mean_of[q]) *
                           rstd_of[q] * (double)gamma[c0 + j] +
                       (double)beta[c0 + j];
      return res ? z + (double)(float)at.row(res, k)[j] : z;
    };
    const unsigned bits = activate<T, V, P, ACT>(a[k], b, res, mean, scale,
                                                 shift, limit, exact);
    store<T, V>(at.row(y, k), a[k]);
    if (ACT == RELU_BITS) *at.template bits<V>(mask, k) = (unsigned char)bits;
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
  auto y = fresh(x.sizes(), x.scalar_type(), x);
  if (stats) *stats = fresh({s.n, s.groups, 2}, torch::kFloat64, x);
  if (x.numel() == 0) return y;
  const void* r = res.defined() ? res.data_ptr() : nullptr;
  const int size = (int)x.element_size();
  const int v = width(s, size, {x.data_ptr(), y.data_ptr(), r});
  const float* gm = gamma.data_ptr<float>();
  const float* bt = beta.data_ptr<float>();
  unsigned char* mk = nullptr;
  if (mask && act == RELU) {
    *mask = fresh({x.numel() / v}, torch::kUInt8, x);
    mk = mask->data_ptr<unsigned char>();
  }
  const hipStream_t stream = cur_stream();
  const int top = fwd_threads(s.cpg % v ? v : 1);
  const Cut slab = cut(s, v, size, top, FWD_VECTORS, false);
  if (slab.threads) {
    TORCH_CHECK(s.n * slab.d.slices * slab.threads < (1L << 32),
                "group_norm: the input is too large");
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
  torch::Tensor own =
      stats ? *stats : fresh({s.n, s.groups, 2}, torch::kFloat64, x);
  int vs = v;       // of the statistics, which may have to be narrower
  const Cut chunk = chop(s, vs, true);
  const Slab& cd = chunk.d;
  const int subs = cd.span * vs == s.cpg ? cd.subs : 1;
  auto part = fresh({s.n * s.groups * subs * cd.chunks, 2}, torch::kFloat64, x);
  int va = v;
  const Cut rows = chop(s, va, false);
  const long all = s.n * s.groups;
  const unsigned joins = (unsigned)std::min<long>(all, 1 << 20);
  const long blocks = s.n * cd.slices * cd.chunks;
  const long applies = s.n * rows.d.slices * rows.d.chunks;
  TORCH_CHECK(std::max(blocks, applies) < (1L << 24),
              "group_norm: the input is too large");
  auto* st = reinterpret_cast<double2*>(own.data_ptr());
  auto* pt = reinterpret_cast<double2*>(part.data_ptr());
  const auto type = x.scalar_type();
  // (a ReLU gives the same values with its bits and without)
  const bool inside = s.cpg % vs == 0, exact = act == RELU;
  with_type(type, vs, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    auto run = [&](auto kernel) {
      kernel<<<(unsigned)blocks, chunk.threads, 0, stream>>>(
          reinterpret_cast<const T*>(x.data_ptr()), pt, cd);
    };
    if (inside && exact) run(stats_kernel<T, V, 1, true>);
    else if (inside) run(stats_kernel<T, V, 1, false>);
    else if (exact) run(stats_kernel<T, V, V, true>);
    else run(stats_kernel<T, V, V, false>);
  });
  const int join = subs * cd.chunks > 64 ? BLOCK : 64;
  join_kernel<<<joins, join, 0, stream>>>(pt, st, all, vs, cd, eps);
  with_type(type, v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    auto run = [&](auto kernel) {
      kernel<<<(unsigned)applies, rows.threads, 0, stream>>>(
          reinterpret_cast<const T*>(x.data_ptr()),
          reinterpret_cast<const T*>(r), reinterpret_cast<T*>(y.data_ptr()),
          mk, st, gm, bt, rows.d);
    };
    with_act(act, mk, [&](auto a) {
      if (s.cpg % v == 0) run(apply_kernel<T, V, 1, decltype(a)::v>);
      else run(apply_kernel<T, V, V, decltype(a)::v>);
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
