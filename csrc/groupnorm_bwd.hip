#include "groupnorm.h"

namespace eg {
namespace gn {

constexpr int SUMS_AT_ONCE = 2, APPLY_AT_ONCE = 4;

// ---- backward -------------------------------------------------------------

// dz / dy of a SiLU at z
__device__ __forceinline__ float silu_slope(float z) {
  const float s = sigmoid(z);
  return s * fmaf(z, 1.f - s, 1.f);
}

// The mean in the kernels has 32 bits, and `low` is what those of 64 are beyond
// it: the same for a whole group, so that the sums are put right once they are
// added, sum dz xh = sum dz (x - mean) rstd - low rstd sum dz, and dx's
//   -rstd s1 - rstd xh s2 = -rstd (s1 - low rstd s2) - rstd^2 s2 (x - mean)
// by what stands in the place of s1.
__device__ __forceinline__ float low_rstd(const double2& st) {
  return (float)((st.x - (float)st.x) * st.y);
}

// A block a group: each channel's sums over the chunks, for dgamma and dbeta,
// and the group's s1, less low rstd s2, and s2.
__global__ void __launch_bounds__(JOIN) bwd_join_kernel(
    const float2* __restrict__ part, const double2* __restrict__ stats,
    const float* __restrict__ gamma,
    float2* __restrict__ channel, float2* __restrict__ group, long groups,
    int per_sample, int cpg, int across, Slab d) {
  // across: threads side by side over channels, a power of two
  __shared__ float2 slot[JOIN];
  __shared__ float sums[JOIN / 64];
  const int lane = threadIdx.x & (across - 1);
  const int share = threadIdx.x / across, shares = blockDim.x / across;
  const float inv = 1.f / ((float)d.hw * (float)cpg);
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const long n = g / per_sample;
    const int c0 = (int)(g % per_sample) * cpg;
    const float low = low_rstd(stats[g]);
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
        s.y = fmaf(-low, s.x, s.y);
        channel[n * d.c + c0 + b + lane] = s;
        s1 = fmaf(gamma[c0 + b + lane], s.x, s1);
        s2 = fmaf(gamma[c0 + b + lane], s.y, s2);
      }
    }
    s1 = add_block(s1, sums);
    s2 = add_block(s2, sums);
    if (threadIdx.x == 0)
      group[g] = make_float2(fmaf(-low, s2, s1) * inv, s2 * inv);
  }
}

// dgamma and dbeta: each channel's sums over the samples, added to what is
// there (a gradient's view in the flat space) or put down. 16 channels, a
// cache line of pairs, by 64 shares of the samples. dgamma and dbeta may be
// one, where gamma and beta are.
constexpr int PC = 16, PN = 64;
__global__ void __launch_bounds__(PC* PN) bwd_params_kernel(
    const float2* __restrict__ channel, float* dgamma, float* dbeta, long n,
    int c, int add) {
  __shared__ Pair slot[PC * PN / 64][PC];
  const int lane = threadIdx.x % PC, share = threadIdx.x / PC;
  const int ch = blockIdx.x * PC + lane;
  Pair s = {0.f, 0.f};
  if (ch < c) {
#pragma unroll 4
    for (long k = share; k < n; k += PN) {
      const float2 e = channel[k * c + ch];
      s += Pair{e.x, e.y};
    }
  }
  s += across<16>(s);
  s += across<32>(s);
  if (threadIdx.x % 64 < PC) slot[threadIdx.x / 64][lane] = s;
  __syncthreads();
  if (threadIdx.x < PC && ch < c) {
    Pair t = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < PC * PN / 64; ++w) t += slot[w][lane];
    dgamma[ch] = add ? dgamma[ch] + t.b : t.b;
    dbeta[ch] = add ? dbeta[ch] + t.a : t.a;
  }
}

// What a thread keeps of its channels, and dz from it. SILU: dz is dy times the
// slope at z; without, it is dy where the forward pass left a bit, or
// everywhere. P: parts of a vector with a mean of their own.
template <typename T, int V, int P, bool SILU_>
struct Channels {
  float mean[P], rstd[P], scale[V], shift[SILU_ ? V : 1];

  __device__ __forceinline__ Channels(const Spot& at, const Slab& d,
                                      const double2* __restrict__ stats,
                                      const float* __restrict__ gamma,
                                      const float* __restrict__ beta) {
    const double2* sample = stats + (long)at.n * d.groups;
    float low[P];
    each_part<P>(at.first, d, [&](int j, int q) {
      const double2 st = sample[q];
      mean[j] = (float)st.x;
      rstd[j] = (float)st.y;
      low[j] = low_rstd(st);
    });
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int p = P == 1 ? 0 : j;
      const float f = gamma[at.first + j];
      scale[j] = f * rstd[p];
      if (SILU_) shift[j] = fmaf(-low[p], f, beta[at.first + j]);
    }
  }

  __device__ __forceinline__ float off(int j, const Vec<T, V>& a) const {
    return a[j] - mean[P == 1 ? 0 : j];
  }

  __device__ __forceinline__ float slope(int j, float off, float r) const {
    return silu_slope(fmaf(off, scale[j], shift[j]) + r);
  }

  // adds a vector to the sums of dz and dz (x - mean), and leaves dz in b
  // where a SiLU makes it
  __device__ __forceinline__ void add(const Vec<T, V>& a, const Vec<T, V>& g,
                                      Vec<T, V>& b, bool res,
                                      float (&s)[2 * V]) const {
    float dz[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float o = off(j, a);
      dz[j] = g[j];
      if (SILU_) dz[j] *= slope(j, o, res ? b[j] : 0.f);
      s[j] += dz[j];
      s[V + j] = fmaf(dz[j], o, s[V + j]);
    }
    if (SILU_) b.put(dz);
  }

  // the block's sums of dz and dz (x - mean) rstd of each channel, in the
  // table's first row
  __device__ __forceinline__ void join(const float (&s)[2 * V], float* table,
                                       const Slab& d) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      table[j * blockDim.x + threadIdx.x] = s[j];
      table[(V + j) * blockDim.x + threadIdx.x] =
          s[V + j] * rstd[P == 1 ? 0 : j];
    }
    __syncthreads();
    fold<2 * V>(table, d, 1);
  }
};

// One vector after the other: the scheduler would else work on all of a
// thread's at once, with registers for as many.
// (A SiLU may have the residual to load for each.)
template <bool SILU_>
__device__ __forceinline__ void in_turn() {
  if (!SILU_) __builtin_amdgcn_sched_barrier(0);
}

template <int V>
__device__ __forceinline__ Pair sums_of(const float* table, int c) {
  return {table[c % V * blockDim.x + c / V],
          table[(V + c % V) * blockDim.x + c / V]};
}

// dx = (rstd gamma) dz - (rstd^2 s2) (x - mean) - rstd s1 (s1 less low rstd
// s2) is two fused multiply-adds of what is fixed for a channel.

// Each channel's sums over one chunk of rows. Bound by vector instructions as
// much as by memory: 4x128x128x320 bf16 with a SiLU, 84 MB in 22 us at some 20
// instructions a value, two of them quarter-rate.
template <typename T, int V, int P, bool SILU_>
__global__ void __launch_bounds__(BLOCK) bwd_sums_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const unsigned char* __restrict__ mask,
    const double2* __restrict__ stats, const float* __restrict__ gamma,
    const float* __restrict__ beta, float2* __restrict__ part, Slab d) {
  __shared__ float table[2 * BLOCK * V];
  const Spot at(d, V);
  const Channels<T, V, P, SILU_> ch(at, d, stats, gamma, beta);
  float s[2 * V] = {};
  each_row<SUMS_AT_ONCE>(at, d, [&](int k) {
    const Vec<T, V> a = load<T, V>(at.row(x, k));
    Vec<T, V> g = load<T, V>(at.row(dy, k)), b;
    if (SILU_ && res) b = load<T, V>(at.row(res, k));
    if (!SILU_ && mask) keep<T, V>(g, *at.template bits<V>(mask, k));
    ch.add(a, g, b, res, s);
  });
  ch.join(s, table, d);
  const int c0 = at.slice * d.lanes * V;
  for (int c = threadIdx.x; c < min(d.lanes * V, d.c - c0); c += blockDim.x) {
    const Pair t = sums_of<V>(table, c);
    part[((long)at.n * d.chunks + at.chunk) * d.c + c0 + c] =
        make_float2(t.a, t.b);
  }
}

// dx and dres from the sums: 4x128x128x320 bf16 with a SiLU, 126 MB in 22.8 us,
// 5.5 TB/s.
template <typename T, int V, int P, bool SILU_>
__global__ void __launch_bounds__(BLOCK) bwd_apply_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const unsigned char* __restrict__ mask,
    const double2* __restrict__ stats, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float2* __restrict__ group,
    T* __restrict__ dx, T* __restrict__ dres, Slab d) {
  const Spot at(d, V);
  const Channels<T, V, P, SILU_> ch(at, d, stats, gamma, beta);
  float by_x[P], less[P];
  each_part<P>(at.first, d, [&](int j, int q) {
    const float2 s = group[(long)at.n * d.groups + q];
    by_x[j] = -ch.rstd[j] * ch.rstd[j] * s.y;
    less[j] = -ch.rstd[j] * s.x;
  });
  each_row<APPLY_AT_ONCE>(at, d, [&](int k) {
    const Vec<T, V> a = load<T, V>(at.row(x, k));
    Vec<T, V> g = load<T, V>(at.row(dy, k)), b, u;
    if (SILU_ && res) b = load<T, V>(at.row(res, k));
    if (!SILU_ && mask) keep<T, V>(g, *at.template bits<V>(mask, k));
    float dz[V], out[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int p = P == 1 ? 0 : j;
      const float o = ch.off(j, a);
      dz[j] = g[j];
      if (SILU_) dz[j] *= ch.slope(j, o, res ? b[j] : 0.f);
      out[j] = fmaf(dz[j], ch.scale[j], fmaf(o, by_x[p], less[p]));
    }
    u.put(out);
    if (SILU_) g.put(dz);
    if (dx) store<T, V>(at.row(dx, k), u);
    if (dres) store<T, V>(at.row(dres, k), g);
  });
}

// All of it in one pass over a slab of whole samples: x and dy stay in
// registers between the sums and dx. 136 MB of 256x32x32x64 bf16 with dres and
// a ReLU's bits in 29 us, 4.7 TB/s; reading the residual and making z
// again, in the place of the bits, took 54.
template <typename T, int V, int I, int P, bool SILU_>
__global__ void __launch_bounds__(SPAN) bwd_slab_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const unsigned char* __restrict__ mask,
    const double2* __restrict__ stats, const float* __restrict__ gamma,
    const float* __restrict__ beta, float2* __restrict__ channel,
    T* __restrict__ dx, T* __restrict__ dres, Slab d) {
  __shared__ float table[2 * SPAN * V];
  __shared__ Pair group[SPAN];
  __shared__ float low_of[SPAN];
  const Spot at(d, V);
  Vec<T, V> a[I], g[I];
  unsigned char bits[I];
#pragma unroll
  for (int k = 0; k < I; ++k) {
    if (at.has(k, d)) {
      a[k] = load<T, V>(at.row(x, k));
      g[k] = load<T, V>(at.row(dy, k));
      if (!SILU_ && mask) bits[k] = *at.template bits<V>(mask, k);
    }
  }
  for (int q = threadIdx.x; q < d.in_slice; q += blockDim.x)
    low_of[q] = low_rstd(
        stats[(long)at.n * d.groups + at.slice * d.in_slice + q]);
  const Channels<T, V, P, SILU_> ch(at, d, stats, gamma, beta);
  float s[2 * V] = {};
#pragma unroll
  for (int k = 0; k < I; ++k) {
    if (at.has(k, d)) {
      Vec<T, V> b;
      if (SILU_ && res) b = load<T, V>(at.row(res, k));
      if (!SILU_ && mask) keep<T, V>(g[k], bits[k]);
      ch.add(a[k], g[k], b, res, s);
      if (dres) store<T, V>(at.row(dres, k), SILU_ ? b : g[k]);
      in_turn<SILU_>();
    }
  }
  ch.join(s, table, d);
  const int width = d.lanes * V;
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    Pair t = sums_of<V>(table, c);
    t.b = fmaf(-low_of[d.by_cpg.of(c)], t.a, t.b);
    const int to = at.slice * width + c;
    channel[(long)at.n * d.c + to] = make_float2(t.a, t.b);
    const float f = gamma[to];
    table[c % V * blockDim.x + c / V] = f * t.a;
    table[(V + c % V) * blockDim.x + c / V] = f * t.b;
  }
  __syncthreads();
  const float inv = 1.f / ((float)d.hw * (float)d.cpg);
  add_groups<Pair>(
      1, d, [&](int e, int) { return sums_of<V>(table, e); },
      [&](int q, const Pair& t) {
        group[q] = Pair{fmaf(-low_of[q], t.b, t.a) * inv, t.b * inv};
      });
  __syncthreads();
  if (!dx || !at.on) return;
  float by_x[P], less[P];
  each_part<P>(at.lane * V, d, [&](int j, int q) {
    by_x[j] = -ch.rstd[j] * ch.rstd[j] * group[q].b;
    less[j] = -ch.rstd[j] * group[q].a;
  });
#pragma unroll
  for (int k = 0; k < I; ++k) {
    if (!at.has(k, d)) break;
    renew<T, V>(a[k]);
    renew<T, V>(g[k]);
    Vec<T, V> b;
    if (SILU_ && res) b = load<T, V>(at.row(res, k));
    float out[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int p = P == 1 ? 0 : j;
      const float o = ch.off(j, a[k]);
      float dz = g[k][j];
      if (SILU_) dz *= ch.slope(j, o, res ? b[j] : 0.f);
      out[j] = fmaf(dz, ch.scale[j], fmaf(o, by_x[p], less[p]));
    }
    a[k].put(out);
    store<T, V>(at.row(dx, k), a[k]);
    in_turn<SILU_>();
  }
}

}  // namespace gn

// dx, the residual's gradient, dgamma and dbeta; an undefined tensor where
// one is not wanted. The parameters' gradients are added to dgamma_out and
// dbeta_out where those are given. mask: a ReLU's bits, res: of a SiLU.
std::vector<torch::Tensor> group_norm_bwd(
    torch::Tensor dy, torch::Tensor x, torch::Tensor stats,
    torch::Tensor gamma, torch::Tensor beta, long groups, long act,
    c10::optional<torch::Tensor> res, c10::optional<torch::Tensor> mask,
    bool want_dx, bool want_dres, c10::optional<torch::Tensor> dgamma_out,
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
  torch::Tensor dx, dres, dgamma, dbeta;
  if (want_dx) dx = fresh(x.sizes(), x.scalar_type(), x);
  if (want_dres) dres = fresh(x.sizes(), x.scalar_type(), x);
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
    dgamma = fresh({s.c}, torch::kFloat32, x);
    dbeta = fresh({s.c}, torch::kFloat32, x);
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
  const int size = (int)x.element_size();
  // the bits are a byte for each vector of the forward pass
  int v = width(s, size, {x.data_ptr(), dy.data_ptr(), r, dxp, drp});
  const unsigned char* mk = nullptr;
  if (act == RELU) {
    TORCH_CHECK(mask && mask->device() == x.device() &&
                    mask->scalar_type() == torch::kUInt8 &&
                    mask->is_contiguous() && mask->numel() > 0 &&
                    x.numel() % mask->numel() == 0,
                "group_norm: mask must be that of the forward pass");
    mk = mask->data_ptr<unsigned char>();
    const int was = (int)(x.numel() / mask->numel());
    if (v < was) dy = dy.clone();      // of lesser alignment than x
    v = was;
    TORCH_CHECK(v <= width(s, size, {x.data_ptr(), dy.data_ptr(), dxp, drp}),
                "group_norm: mask must be that of the forward pass");
  }
  const auto* st = reinterpret_cast<const double2*>(stats.data_ptr());
  const float* gm = gamma.data_ptr<float>();
  const float* bt = beta.data_ptr<float>();
  const hipStream_t stream = cur_stream();
  auto channel = fresh({s.n, s.c, 2}, torch::kFloat32, x);
  auto* cp = reinterpret_cast<float2*>(channel.data_ptr());
  auto params = [&] {
    bwd_params_kernel<<<ceil_div(s.c, PC), PC * PN, 0, stream>>>(
        cp, dgamma.data_ptr<float>(), dbeta.data_ptr<float>(), s.n, s.c,
        add ? 1 : 0);
  };
  const Cut slab = cut(s, v, size, SPAN, BWD_VECTORS, true);
  if (slab.threads) {
    TORCH_CHECK(s.n * slab.d.slices * slab.threads < (1L << 32),
                "group_norm: the input is too large");
    with_slab(x.scalar_type(), v, slab.vectors, s.cpg % v == 0, [&](auto tag) {
      using G = decltype(tag);
      using T = typename G::type;
      if constexpr (G::i <= BWD_VECTORS) {
        const unsigned blocks = (unsigned)(s.n * slab.d.slices);
        auto run = [&](auto kernel) {
          kernel<<<blocks, slab.threads, 0, stream>>>(
              reinterpret_cast<const T*>(dy.data_ptr()),
              reinterpret_cast<const T*>(x.data_ptr()),
              reinterpret_cast<const T*>(r), mk, st, gm, bt, cp,
              reinterpret_cast<T*>(dxp), reinterpret_cast<T*>(drp), slab.d);
        };
        if (act == SILU) run(bwd_slab_kernel<T, G::v, G::i, G::p, true>);
        else run(bwd_slab_kernel<T, G::v, G::i, G::p, false>);
      }
    });
    params();
    return {dx, dres, dgamma, dbeta};
  }
  const Cut chunk = chop(s, v, false);
  const Slab& cd = chunk.d;
  const long blocks = s.n * cd.slices * cd.chunks;
  TORCH_CHECK(blocks < (1L << 24), "group_norm: the input is too large");
  auto part = fresh({s.n, cd.chunks, s.c, 2}, torch::kFloat32, x);
  auto group = fresh({s.n, groups, 2}, torch::kFloat32, x);
  auto* pt = reinterpret_cast<float2*>(part.data_ptr());
  auto* gp = reinterpret_cast<float2*>(group.data_ptr());
  const auto type = x.scalar_type();
  const bool inside = s.cpg % v == 0;
  with_type(type, v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    auto sums = [&](auto kernel) {
      kernel<<<(unsigned)blocks, chunk.threads, 0, stream>>>(
          reinterpret_cast<const T*>(dy.data_ptr()),
          reinterpret_cast<const T*>(x.data_ptr()),
          reinterpret_cast<const T*>(r), mk, st, gm, bt, pt, cd);
    };
    if (inside && act == SILU) sums(bwd_sums_kernel<T, V, 1, true>);
    else if (inside) sums(bwd_sums_kernel<T, V, 1, false>);
    else if (act == SILU) sums(bwd_sums_kernel<T, V, V, true>);
    else sums(bwd_sums_kernel<T, V, V, false>);
  });
  // a block for each group, of about four entries a thread
  const long all = s.n * groups;
  const unsigned joins = (unsigned)std::min<long>(all, 1 << 20);
  int across = 1, join = 64;
  while (across < s.cpg && across < JOIN) across *= 2;
  while (join < JOIN && (join < across || 4L * join < (long)s.cpg * cd.chunks))
    join *= 2;
  bwd_join_kernel<<<joins, join, 0, stream>>>(pt, st, gm, cp, gp, all, s.groups,
                                              s.cpg, across, cd);
  params();
  if (!dxp && !drp) return {dx, dres, dgamma, dbeta};
  with_type(type, v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    auto apply = [&](auto kernel) {
      kernel<<<(unsigned)blocks, chunk.threads, 0, stream>>>(
          reinterpret_cast<const T*>(dy.data_ptr()),
          reinterpret_cast<const T*>(x.data_ptr()),
          reinterpret_cast<const T*>(r), mk, st, gm, bt, gp,
          reinterpret_cast<T*>(dxp), reinterpret_cast<T*>(drp), cd);
    };
    if (inside && act == SILU) apply(bwd_apply_kernel<T, V, 1, true>);
    else if (inside) apply(bwd_apply_kernel<T, V, 1, false>);
    else if (act == SILU) apply(bwd_apply_kernel<T, V, V, true>);
    else apply(bwd_apply_kernel<T, V, V, false>);
  });
  return {dx, dres, dgamma, dbeta};
}

}  // namespace eg
