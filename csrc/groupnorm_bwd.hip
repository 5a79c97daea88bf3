#include "groupnorm.h"

namespace eg {
namespace gn {

// ---- backward -------------------------------------------------------------

// What a thread keeps of its V channels. SILU: dz is dy times the slope at z;
// without, it is dy where the forward pass left a bit, or everywhere.
template <typename T, int V, bool SILU_>
struct Channels {
  float mean[V], rstd[V], gamma[V], beta[SILU_ ? V : 1];

  __device__ __forceinline__ Channels(const double2* sample, int c0,
                                      const float* g, const float* b,
                                      int cpg) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double2 st = sample[(c0 + j) / cpg];
      mean[j] = (float)st.x;
      rstd[j] = (float)st.y;
      gamma[j] = g[c0 + j];
      if (SILU_) beta[j] = b[c0 + j];
    }
  }

  __device__ __forceinline__ float dz(int j, float xh, float r,
                                      float dy) const {
    if (!SILU_) return dy;
    const float z = fmaf(xh, gamma[j], beta[j]) + r;
    const float s = sigmoid(z);
    return dy * (s * fmaf(z, 1.f - s, 1.f));
  }
};

// Each channel's sums of dz and of dz xh over one chunk of rows.
template <typename T, int V, bool SILU_>
__global__ void __launch_bounds__(BLOCK) bwd_sums_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const unsigned char* __restrict__ mask,
    const double2* __restrict__ stats, const float* __restrict__ gamma,
    const float* __restrict__ beta, float2* __restrict__ part, int groups,
    int cpg, Deal d) {
  __shared__ float slot[BLOCK / 2 * 2 * V];
  const Place at(d);
  float sums[2 * V] = {};
  if (at.on) {
    const Channels<T, V, SILU_> ch(stats + (long)at.n * groups, at.col * V,
                                   gamma, beta, cpg);
    const long base = ((long)at.n * d.hw + at.begin) * d.c + at.col * V;
#pragma unroll 2
    for (int k = at.r; k < at.count; k += d.rows) {
      const long i = base + (long)k * d.c;
      const Vec<T, V> a = load<T, V>(x + i);
      Vec<T, V> g = load<T, V>(dy + i), b;
      if (SILU_ && res) b = load<T, V>(res + i);
      if (!SILU_ && mask) keep<T, V>(g, mask[i / V]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = ((float)a.v[j] - ch.mean[j]) * ch.rstd[j];
        const float dz = ch.dz(j, xh, SILU_ && res ? (float)b.v[j] : 0.f,
                               (float)g.v[j]);
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
__global__ void __launch_bounds__(JOIN) bwd_join_kernel(
    const float2* __restrict__ part, const float* __restrict__ gamma,
    float2* __restrict__ channel, float2* __restrict__ group, long groups,
    int per_sample, int cpg, int across, Deal d) {
  // across: threads side by side over channels, a power of two
  __shared__ float2 slot[JOIN];
  __shared__ float sums[JOIN / 64];
  const int lane = threadIdx.x % across, share = threadIdx.x / across;
  const int shares = JOIN / across;
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
// there (a gradient's view in the flat space) or put down. 16 channels, a
// cache line of pairs, by 64 shares of the samples.
constexpr int PC = 16, PN = 64;
__global__ void __launch_bounds__(PC* PN) bwd_params_kernel(
    const float2* __restrict__ channel, float* __restrict__ dgamma,
    float* __restrict__ dbeta, long n, int c, int add) {
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
  s += across(s, 16);
  s += across(s, 32);
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

template <typename T, int V, bool SILU_>
__global__ void __launch_bounds__(BLOCK) bwd_apply_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const unsigned char* __restrict__ mask,
    const double2* __restrict__ stats, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float2* __restrict__ group,
    T* __restrict__ dx, T* __restrict__ dres, int groups, int cpg, Deal d) {
  const Place at(d);
  if (!at.on) return;
  const Channels<T, V, SILU_> ch(stats + (long)at.n * groups, at.col * V,
                                 gamma, beta, cpg);
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
    const Vec<T, V> a = load<T, V>(x + i);
    Vec<T, V> g = load<T, V>(dy + i), b, u;
    if (SILU_ && res) b = load<T, V>(res + i);
    if (!SILU_ && mask) keep<T, V>(g, mask[i / V]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float xh = ((float)a.v[j] - ch.mean[j]) * ch.rstd[j];
      const float dz = ch.dz(j, xh, SILU_ && res ? (float)b.v[j] : 0.f,
                             (float)g.v[j]);
      u.v[j] = (T)(ch.rstd[j] *
                   (fmaf(dz, ch.gamma[j], -s1[j]) - xh * s2[j]));
      if (SILU_) g.v[j] = (T)dz;
    }
    if (dx) store<T, V>(dx + i, u);
    if (dres) store<T, V>(dres + i, g);
  }
}

// The slab in one pass: x and dy stay in registers between the sums and dx.
template <typename T, int V, int I, int P, bool SILU_>
__global__ void __launch_bounds__(SLAB) bwd_slab_kernel(
    const T* __restrict__ dy, const T* __restrict__ x,
    const T* __restrict__ res, const unsigned char* __restrict__ mask,
    const double2* __restrict__ stats, const float* __restrict__ gamma,
    const float* __restrict__ beta, float2* __restrict__ channel,
    T* __restrict__ dx, T* __restrict__ dres, Slab d) {
  __shared__ Pair table[SLAB * V];
  __shared__ Pair group[SLAB];
  const Spot at(d, V);
  const long base = (long)at.n * d.hw * d.c + at.first + at.lane * V;
  Vec<T, V> a[I], g[I];
  unsigned bits[I];
#pragma unroll
  for (int k = 0; k < I; ++k) {
    const int row = at.r + k * d.rows;
    if (at.on && row < d.hw) {
      const long i = base + (long)row * d.c;
      a[k] = load<T, V>(x + i);
      g[k] = load<T, V>(dy + i);
      if (!SILU_ && mask) bits[k] = mask[i / V];
    }
  }
  // mean, rstd, s1 and s2 of a thread's channels: one, or P
  const double2* sample = stats + (long)at.n * d.groups;
  const int c0 = at.on ? at.first + at.lane * V : 0;
  float mean[P], rstd[P], gam[V], bet[SILU_ ? V : 1];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const double2 st = sample[(c0 + j) / d.cpg];
    mean[j] = (float)st.x;
    rstd[j] = (float)st.y;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    gam[j] = gamma[c0 + j];
    if (SILU_) bet[j] = beta[c0 + j];
  }
  auto slope = [&](int j, float off, float r) {
    const float z = fmaf(off * rstd[P == 1 ? 0 : j], gam[j], bet[j]) + r;
    const float s = sigmoid(z);
    return s * fmaf(z, 1.f - s, 1.f);
  };
  // sums of dz and of dz (x - mean); the latter's rstd comes at the end
  float s[2 * V] = {};
#pragma unroll
  for (int k = 0; k < I; ++k) {
    const int row = at.r + k * d.rows;
    if (at.on && row < d.hw) {
      const long i = base + (long)row * d.c;
      Vec<T, V> b;
      if (SILU_ && res) b = load<T, V>(res + i);
      if (!SILU_ && mask) keep<T, V>(g[k], bits[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float off = (float)a[k].v[j] - mean[P == 1 ? 0 : j];
        float dz = (float)g[k].v[j];
        if (SILU_) {
          dz *= slope(j, off, res ? (float)b.v[j] : 0.f);
          b.v[j] = (T)dz;
        }
        s[j] += dz;
        s[V + j] = fmaf(dz, off, s[V + j]);
      }
      if (dres) store<T, V>(dres + i, SILU_ ? b : g[k]);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    table[threadIdx.x * V + j] =
        Pair{s[j], s[V + j] * rstd[P == 1 ? 0 : j]};
  __syncthreads();
  // rows of a channel: first in `parts` shares, in place, then those
  const int width = d.lanes * V;
  const int parts = max(1, (int)blockDim.x / width);
  for (int u = threadIdx.x; u < width * parts; u += blockDim.x) {
    const int c = u % width, p = u / width;
    Pair t = {0.f, 0.f};
    for (int row = p; row < d.rows; row += parts) t += table[row * width + c];
    if (p < d.rows) table[u] = t;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    Pair t = table[c];
    for (int p = 1; p < min(parts, d.rows); ++p) t += table[p * width + c];
    const int to = at.first + c;
    channel[(long)at.n * d.c + to] = make_float2(t.a, t.b);
    const float f = gamma[to];
    table[c] = Pair{f * t.a, f * t.b};
  }
  __syncthreads();
  const float inv = 1.f / ((float)d.hw * (float)d.cpg);
  add_groups<Pair>(table, 1, d.cpg, d, [&](int q, const Pair& t) {
    group[q] = Pair{t.a * inv, t.b * inv};
  });
  __syncthreads();
  if (!dx || !at.on) return;
  // dx = (rstd gamma) dz - (rstd^2 s2) (x - mean) - rstd s1
  float by_x[P], less[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const Pair t = group[(at.lane * V + j) / d.cpg];
    by_x[j] = -rstd[j] * rstd[j] * t.b;
    less[j] = -rstd[j] * t.a;
  }
#pragma unroll
  for (int k = 0; k < I; ++k) {
    const int row = at.r + k * d.rows;
    if (row >= d.hw) break;
    const long i = base + (long)row * d.c;
    Vec<T, V> b;
    if (SILU_ && res) b = load<T, V>(res + i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int p = P == 1 ? 0 : j;
      const float off = (float)a[k].v[j] - mean[p];
      float dz = (float)g[k].v[j];
      if (SILU_) dz *= slope(j, off, res ? (float)b.v[j] : 0.f);
      a[k].v[j] = (T)fmaf(dz, gam[j] * rstd[p], fmaf(off, by_x[p], less[p]));
    }
    store<T, V>(dx + i, a[k]);
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
    auto both = torch::empty({2, s.c}, f32);
    dgamma = both[0];
    dbeta = both[1];
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
  auto channel = torch::empty({s.n, s.c, 2}, f32);
  auto* cp = reinterpret_cast<float2*>(channel.data_ptr());
  auto params = [&] {
    bwd_params_kernel<<<ceil_div(s.c, PC), PC * PN, 0, stream>>>(
        cp, dgamma.data_ptr<float>(), dbeta.data_ptr<float>(), s.n, s.c,
        add ? 1 : 0);
  };
  const Cut slab = cut(s, v, size, BWD_VECTORS);
  if (slab.threads) {
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
  const Deal d = deal(s.hw, s.c, v, s.n);
  auto part = torch::empty({s.n, d.chunks, s.c, 2}, f32);
  auto group = torch::empty({s.n, groups, 2}, f32);
  const dim3 grid((unsigned)(s.n * d.chunks), 1,
                  (unsigned)((d.cols + d.lanes - 1) / d.lanes));
  const long all = s.n * groups;
  const unsigned joins = (unsigned)std::min<long>(all, 1 << 20);
  auto* pt = reinterpret_cast<float2*>(part.data_ptr());
  auto* gp = reinterpret_cast<float2*>(group.data_ptr());
  int across = 1;
  while (across < s.cpg && across < JOIN) across *= 2;
  with_type(x.scalar_type(), v, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int V = decltype(tag)::v;
    const T* xp = reinterpret_cast<const T*>(x.data_ptr());
    const T* yp = reinterpret_cast<const T*>(dy.data_ptr());
    const T* rp = reinterpret_cast<const T*>(r);
    auto sums = [&](auto kernel) {
      kernel<<<grid, BLOCK, 0, stream>>>(yp, xp, rp, mk, st, gm, bt, pt,
                                         s.groups, s.cpg, d);
    };
    auto apply = [&](auto kernel) {
      kernel<<<grid, BLOCK, 0, stream>>>(
          yp, xp, rp, mk, st, gm, bt, gp, reinterpret_cast<T*>(dxp),
          reinterpret_cast<T*>(drp), s.groups, s.cpg, d);
    };
    if (act == SILU) sums(bwd_sums_kernel<T, V, true>);
    else sums(bwd_sums_kernel<T, V, false>);
    bwd_join_kernel<<<joins, JOIN, 0, stream>>>(
        pt, gm, cp, gp, all, s.groups, s.cpg, across, d);
    params();
    if (dxp || drp) {
      if (act == SILU) apply(bwd_apply_kernel<T, V, true>);
      else apply(bwd_apply_kernel<T, V, false>);
    }
  });
  return {dx, dres, dgamma, dbeta};
}

}  // namespace eg
