// AdamW over every tensor of the flat space at once, with the moments held
// in 32 or in 8 bits, and each tensor's squared norm for the trigger.
//
//   m' = b1 m + (1 - b1) g            v' = b2 v + (1 - b2) g^2
//   p' = p - lr wd p - lr (m' / (1 - b1^t)) / (sqrt(v' / (1 - b2^t)) + eps)
//   sq[i] = sum of p'^2 over tensor i
//
// The flat space is cut into chunks that never cross a tensor, so a block
// has one decay and one norm. Each block leaves its part of the norm in a
// slot of its own, and a second kernel adds the slots in a fixed order: the
// norms, and with them the trigger's decisions, are the same on every run.
// The step count, the learning rate and the bias corrections live on the
// device, where the second kernel moves them on: a captured step counts
// right on every replay.
//
// 8-bit moments. 64 values share one power of two, 2^(E-127), kept in a byte:
// the one that leaves the largest of them below 2 once it is rounded up. Each
// value is a byte on top of it: m has a sign, 4 bits of exponent and 3 behind
// the leading one (2^-17 to 1.875), v has no sign and 5 bits of exponent
// (2^-33 to 1.875). Values are rounded up with the probability of what lies
// below the grid, from 16 hashed bits of (seed, step, place): with b2 = 0.999
// a step moves v by a thousandth of itself, which rounding to the nearest of
// 8 steps an octave would always take back. A v above zero stays above zero,
// since m / sqrt(v) would blow up. A block with a value that is not finite
// has E = 255 and stands for NaN throughout. E is at least 18 (m) and 34 (v):
// every value is then a normal number in bfloat16, which holds it exactly.

// What bounds it is memory. 17.4 M weights: 28 bytes each in 72 us, 6.8 TB/s,
// with 32 bits; 16 1/16 bytes each in 48 us, 5.8 TB/s, with 8. Four values a
// thread, so that 16 lanes are a block of 64 and its largest value is found
// without shared memory.

#include "common.h"

#include <c10/core/DeviceGuard.h>

namespace eg {
namespace adamw {

constexpr int BLOCK = 256;
constexpr int QB = 64;          // values that share an exponent
constexpr unsigned INF_BITS = 0x7f800000u;

// coef: [lr, 1 / (1 - b1^t), 1 / sqrt(1 - b2^t)] of the step to come
struct Hyper {
  float b1, c1, b2, c2, eps;    // c = 1 - b
  unsigned seed;
};

// m' and v' are rounded after each operation, as elementwise tensor
// operations round them, so that a code never hangs on the compiler's choice
// of a fused multiply-add.
__device__ __forceinline__ float ema(float s, float b, float x, float c) {
#pragma clang fp contract(off)
  float a = s * b;
  float d = x * c;
  return a + d;
}

__device__ __forceinline__ float square(float x) {
#pragma clang fp contract(off)
  return x * x;
}

// The hardware's root and reciprocal, off by a step or two: 2^-22 of an
// update. A root takes a v below 2^-126 for 0, 1e-19 off; eps is 1e-12 at
// least. (With the exact ones the 8-bit step of 17.4 M weights took 65 us.)
__device__ __forceinline__ float stepped(float p, float m, float v, float k1,
                                         float k2, float eps, float decay) {
  const float denom = fmaf(__builtin_amdgcn_sqrtf(v), k2, eps);
  return fmaf(decay, p, p) + k1 * m * __builtin_amdgcn_rcpf(denom);
}

// ---- the 8-bit grid -------------------------------------------------------

template <int EXP_BITS>
__device__ __forceinline__ int shared_exponent(unsigned top) {
  int e = (int)((top + 0xfffffu) >> 23);
  e = min(max(e, 2 + (1 << EXP_BITS)), 254);
  return top >= INF_BITS ? 255 : e;
}

// 2^(e - 127), NaN for 255
__device__ __forceinline__ float power(int e) {
  return __uint_as_float(e == 255 ? 0x7fc00000u : (unsigned)e << 23);
}

// y = |x| 2^(127 - e) as a byte; `random` has 16 bits
template <int EXP_BITS>
__device__ __forceinline__ unsigned encode(float y, unsigned random) {
  constexpr int BIAS = (1 << EXP_BITS) - 1;     // of the byte's own exponent
  const unsigned normal = ((__float_as_uint(y) + (random << 4)) >> 20) -
                          (unsigned)((127 - BIAS) << 3);
  // below the smallest normal: a multiple of 2^(-2 - BIAS), 16 bits further
  constexpr float STEPS = BIAS == 15 ? 0x1p33f : 0x1p49f;
  constexpr float LEAST = BIAS == 15 ? 0x1p-14f : 0x1p-30f;
  const unsigned low = ((unsigned)(y * STEPS) + random) >> 16;
  return min(y < LEAST ? low : normal, (unsigned)((8 << EXP_BITS) - 1));
}

// byte J of four, without its power of two. The byte's exponent and the bits
// behind it go where a float's are: a float's subnormals are then the byte's,
// and one exact product sets the exponent right.
template <int J>
__device__ __forceinline__ float decode_m(unsigned code) {
  const unsigned up = code << (24 - 8 * J);
  const unsigned bits = (up >> 4 & 0x07f00000u) | (up & 0x80000000u);
  return __uint_as_float(bits) * 0x1p112f;
}

template <int J>
__device__ __forceinline__ float decode_v(unsigned code) {
  return __uint_as_float((code >> (8 * J) & 255u) << 20) * 0x1p96f;
}

__device__ __forceinline__ void decode4(uint2 code, uchar2 e, float* m,
                                        float* v) {
  const float pm = power(e.x), pv = power(e.y);
  m[0] = decode_m<0>(code.x) * pm;
  m[1] = decode_m<1>(code.x) * pm;
  m[2] = decode_m<2>(code.x) * pm;
  m[3] = decode_m<3>(code.x) * pm;
  v[0] = decode_v<0>(code.y) * pv;
  v[1] = decode_v<1>(code.y) * pv;
  v[2] = decode_v<2>(code.y) * pv;
  v[3] = decode_v<3>(code.y) * pv;
}

// the largest of 16 lanes in all of them: within fours, eights, sixteens
__device__ __forceinline__ unsigned max16(unsigned v) {
  auto step = [](unsigned a, auto ctrl) {
    return max(a, (unsigned)__builtin_amdgcn_update_dpp(
                      0, (int)a, decltype(ctrl)::value, 0xf, 0xf, false));
  };
  v = step(v, std::integral_constant<int, 0xb1>());    // quad: 1 0 3 2
  v = step(v, std::integral_constant<int, 0x4e>());    // quad: 2 3 0 1
  v = step(v, std::integral_constant<int, 0x141>());   // mirror of 8
  return step(v, std::integral_constant<int, 0x140>());   // mirror of 16
}

// ---- the step -------------------------------------------------------------

// what the end of a step needs: the tensors' chunks and norms, b1^t and b2^t
struct Finish {
  const long* first;
  float* norms;
  double* powers;
  unsigned* count;    // blocks that have ended
  int tensors;
  double b1, b2;
};

__device__ __forceinline__ void next_step(const Finish& end, float* coef,
                                          long* step) {
  const double p1 = end.powers[0] * end.b1, p2 = end.powers[1] * end.b2;
  step[0] += 1;
  end.powers[0] = p1;
  end.powers[1] = p2;
  coef[1] = (float)(1.0 / (1.0 - p1));
  coef[2] = (float)(1.0 / sqrt(1.0 - p2));
}

// Gradients and moments pass by: nothing reads them again before the next
// step, and kept out of the caches they leave room for the weights, which the
// next pass reads. On 17.4 M weights the 32-bit step takes 72 us so, and 91 us
// without; the 8-bit step 52 and 56.
template <typename T>
__device__ __forceinline__ T pass_in(const T* p) {
  static_assert(sizeof(T) == 16 || sizeof(T) == 8, "");
  using W = std::conditional_t<sizeof(T) == 16, f32x4, unsigned long>;
  const W w = __builtin_nontemporal_load(reinterpret_cast<const W*>(p));
  T t;
  __builtin_memcpy(&t, &w, sizeof(T));
  return t;
}

template <typename T>
__device__ __forceinline__ void pass_out(T* p, const T& t) {
  using W = std::conditional_t<sizeof(T) == 16, f32x4, unsigned long>;
  W w;
  __builtin_memcpy(&w, &t, sizeof(T));
  __builtin_nontemporal_store(w, reinterpret_cast<W*>(p));
}

// chunks: [start, length, tensor] each; a chunk starts at a multiple of QB
// and is taken to the next one beyond its length: the gap behind a tensor
// belongs to it, and zeros there stay zeros.
//
// JOINED: the grid is at most BLOCK blocks, and the one that ends last adds
// the norms up and moves the step on, in the place of a second launch (27,480
// weights: 8.9 us in two, 5.5 in one). Each block's part is released before it
// counts itself, and the last has acquired them all once it has counted.
template <int BITS, bool JOINED>
__global__ void __launch_bounds__(BLOCK) step_kernel(
    float* __restrict__ param, const float* __restrict__ grad,
    float* __restrict__ m32, float* __restrict__ v32,
    uint2* __restrict__ codes, uchar2* __restrict__ exps,
    const long* __restrict__ chunks, const float* __restrict__ decay,
    float* coef, long* step, float* part, Hyper h, Finish end) {
  const long start = chunks[3 * blockIdx.x];
  const int len = (int)chunks[3 * blockIdx.x + 1];
  const long tensor = chunks[3 * blockIdx.x + 2];
  const float lr = coef[0], k1 = -lr * coef[1], k2 = coef[2];
  const float shrink = -lr * decay[tensor];
  const unsigned key = hash_u32(h.seed, (unsigned)(step[0] + 1));
  const int padded = (len + QB - 1) / QB * QB;
  float acc = 0.f;
  for (int i = threadIdx.x * 4; i < padded; i += BLOCK * 4) {
    const long at = start + i;
    float4 p = *reinterpret_cast<const float4*>(param + at);
    const float4 g = pass_in(reinterpret_cast<const float4*>(grad + at));
    float4 m, v;
    float* pp = reinterpret_cast<float*>(&p);
    const float* gg = reinterpret_cast<const float*>(&g);
    float* mm = reinterpret_cast<float*>(&m);
    float* vv = reinterpret_cast<float*>(&v);
    if (BITS == 32) {
      m = pass_in(reinterpret_cast<const float4*>(m32 + at));
      v = pass_in(reinterpret_cast<const float4*>(v32 + at));
    } else {
      decode4(pass_in(codes + (at >> 2)), exps[at / QB], mm, vv);
    }
    unsigned top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mm[j] = ema(mm[j], h.b1, gg[j], h.c1);
      vv[j] = ema(vv[j], h.b2, square(gg[j]), h.c2);
      pp[j] = stepped(pp[j], mm[j], vv[j], k1, k2, h.eps, shrink);
      if (i + j < len) acc = fmaf(pp[j], pp[j], acc);
      top_m = max(top_m, __float_as_uint(mm[j]) & 0x7fffffffu);
      top_v = max(top_v, __float_as_uint(vv[j]) & 0x7fffffffu);
    }
    *reinterpret_cast<float4*>(param + at) = p;
    if (BITS == 32) {
      pass_out(reinterpret_cast<float4*>(m32 + at), m);
      pass_out(reinterpret_cast<float4*>(v32 + at), v);
    } else {
      // 16 lanes hold one block of 64, and all of them are here: chunks are
      // cut and padded in whole blocks
      const int em = shared_exponent<4>(max16(top_m));
      const int ev = shared_exponent<5>(max16(top_v));
      uint2 code = {0u, 0u};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned long place = (unsigned long)(at + j);
        const unsigned r =
            hash_u32(key + (unsigned)(place >> 32), (unsigned)place);
        unsigned qm = encode<4>(ldexpf(fabsf(mm[j]), 127 - em), r & 0xffffu);
        qm |= __float_as_uint(mm[j]) >> 24 & 128u;
        unsigned qv = encode<5>(ldexpf(vv[j], 127 - ev), r >> 16);
        qv = max(qv, vv[j] > 0.f ? 1u : 0u);
        code.x |= qm << (8 * j);
        code.y |= qv << (8 * j);
      }
      pass_out(codes + (at >> 2), code);
      if ((threadIdx.x & 15) == 0)
        exps[at / QB] = make_uchar2((unsigned char)em, (unsigned char)ev);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) acc += __shfl_xor(acc, d);
  __shared__ float waves[BLOCK / 64];
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = acc;
  __syncthreads();
  __shared__ bool last;
  if (threadIdx.x == 0) {
    float s = 0.f;
    for (int w = 0; w < BLOCK / 64; ++w) s += waves[w];
    part[blockIdx.x] = s;
    if (JOINED) {
      __threadfence();
      last = atomicAdd(end.count, 1u) == gridDim.x - 1;
      __threadfence();
    }
  }
  if (!JOINED) return;
  __syncthreads();
  if (!last) return;
  __shared__ float parts[BLOCK];
  if (threadIdx.x < gridDim.x)
    parts[threadIdx.x] = __hip_atomic_load(part + threadIdx.x,
                                           __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (int i = threadIdx.x; i < end.tensors; i += BLOCK) {
    float s = 0.f;
#pragma unroll 8
    for (long k = end.first[i]; k < end.first[i + 1]; ++k) s += parts[k];
    end.norms[i] = s;
  }
  if (threadIdx.x == 0) {
    *end.count = 0;
    next_step(end, coef, step);
  }
}

// One block a tensor: its chunks' parts, added in a fixed order. The first
// block moves the step on.
constexpr int FINISH = 512;
__global__ void __launch_bounds__(FINISH) finish_kernel(
    const float* __restrict__ part, float* coef, long* step, Finish end) {
  const long a = end.first[blockIdx.x], b = end.first[blockIdx.x + 1];
  float acc = 0.f;
#pragma unroll 8
  for (long i = a + threadIdx.x; i < b; i += FINISH) acc += part[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) acc += __shfl_xor(acc, d);
  __shared__ float waves[FINISH / 64];
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    float s = 0.f;
    for (int w = 0; w < FINISH / 64; ++w) s += waves[w];
    end.norms[blockIdx.x] = s;
    if (blockIdx.x == 0) next_step(end, coef, step);
  }
}

__global__ void __launch_bounds__(BLOCK) moments_kernel(
    const uint2* __restrict__ codes, const uchar2* __restrict__ exps,
    bf16x4* __restrict__ m, bf16x4* __restrict__ v, long quads) {
  const long stride = (long)gridDim.x * BLOCK;
  for (long i = (long)blockIdx.x * BLOCK + threadIdx.x; i < quads;
       i += stride) {
    float x[4], y[4];
    decode4(codes[i], exps[i / (QB / 4)], x, y);
    bf16x4 a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = (__bf16)x[j];
      b[j] = (__bf16)y[j];
    }
    m[i] = a;
    v[i] = b;
  }
}

static void check(const torch::Tensor& t, const char* name,
                  c10::ScalarType type, long numel,
                  const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name,
              " must be on the parameters' GPU");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ",
              t.scalar_type());
  TORCH_CHECK(t.numel() == numel, name, " must have ", numel,
              " elements, got ", t.numel());
}

}  // namespace adamw

// codes: for each 4 values 4 bytes of m, then 4 of v; exps: for each 64 the
// exponents of m and of v. Where they are empty the moments are m and v in
// fp32. chunks [k, 3] lists each tensor's chunks in turn, first[i] is the
// place of tensor i's first chunk; both are the caller's plan, made for
// param's layout. coef and powers (b1^t, b2^t) are those of the step to come.
// part [k + 1] is scratch that goes with the moments, zero at first.
torch::Tensor adamw_step_norm(torch::Tensor param, torch::Tensor grad,
                              torch::Tensor m, torch::Tensor v,
                              torch::Tensor codes, torch::Tensor exps,
                              torch::Tensor chunks, torch::Tensor first,
                              torch::Tensor decay, torch::Tensor coef,
                              torch::Tensor powers, torch::Tensor step,
                              torch::Tensor part, double b1, double b2,
                              double eps, long seed) {
  using namespace adamw;
  CHECK_IN(param);
  TORCH_CHECK(eps >= 1e-12, "eps must be at least 1e-12");
  TORCH_CHECK(param.scalar_type() == torch::kFloat32, "param must be fp32");
  const long n = param.numel();
  TORCH_CHECK(n % QB == 0, "the flat space must be padded to ", QB);
  TORCH_CHECK((reinterpret_cast<uintptr_t>(param.data_ptr()) |
               reinterpret_cast<uintptr_t>(grad.data_ptr())) % 16 == 0,
              "param and grad must be 16-byte aligned");
  const bool bits8 = codes.numel() > 0;
  check(grad, "grad", torch::kFloat32, n, param);
  if (bits8) {
    check(codes, "codes", torch::kUInt8, 2 * n, param);
    check(exps, "exps", torch::kUInt8, 2 * (n / QB), param);
  } else {
    check(m, "m", torch::kFloat32, n, param);
    check(v, "v", torch::kFloat32, n, param);
  }
  const long sz = decay.numel(), k = chunks.numel() / 3;
  check(chunks, "chunks", torch::kInt64, 3 * k, param);
  check(first, "first", torch::kInt64, sz + 1, param);
  check(decay, "decay", torch::kFloat32, sz, param);
  check(coef, "coef", torch::kFloat32, 3, param);
  check(powers, "powers", torch::kFloat64, 2, param);
  check(step, "step", torch::kInt64, 1, param);
  check(part, "part", torch::kFloat32, k + 1, param);
  const c10::DeviceGuard guard(param.device());
  auto norms = torch::empty({sz}, param.options());
  if (sz == 0) return norms;
  const Hyper h{(float)b1, (float)(1.0 - b1), (float)b2, (float)(1.0 - b2),
                (float)eps, (unsigned)seed};
  const Finish end{first.data_ptr<long>(), norms.data_ptr<float>(),
                   powers.data_ptr<double>(),
                   reinterpret_cast<unsigned*>(part.data_ptr<float>() + k),
                   (int)sz, b1, b2};
  const hipStream_t stream = cur_stream();
  auto run = [&](auto kernel) {
    kernel<<<(unsigned)k, BLOCK, 0, stream>>>(
        param.data_ptr<float>(), grad.data_ptr<float>(),
        bits8 ? nullptr : m.data_ptr<float>(),
        bits8 ? nullptr : v.data_ptr<float>(),
        bits8 ? reinterpret_cast<uint2*>(codes.data_ptr()) : nullptr,
        bits8 ? reinterpret_cast<uchar2*>(exps.data_ptr()) : nullptr,
        chunks.data_ptr<long>(), decay.data_ptr<float>(),
        coef.data_ptr<float>(), step.data_ptr<long>(),
        part.data_ptr<float>(), h, end);
  };
  const bool joined = k > 0 && k <= BLOCK;
  if (joined) {
    if (bits8) run(step_kernel<8, true>); else run(step_kernel<32, true>);
    return norms;
  }
  if (k) {
    if (bits8) run(step_kernel<8, false>); else run(step_kernel<32, false>);
  }
  finish_kernel<<<(unsigned)sz, FINISH, 0, stream>>>(
      part.data_ptr<float>(), coef.data_ptr<float>(), step.data_ptr<long>(),
      end);
  return norms;
}

// the values that 8-bit moments stand for, exact in bfloat16
std::vector<torch::Tensor> adamw_moments(torch::Tensor codes,
                                         torch::Tensor exps) {
  using namespace adamw;
  CHECK_IN(codes);
  const long n = codes.numel() / 2;
  TORCH_CHECK(n % QB == 0 && codes.numel() == 2 * n, "codes must hold whole "
              "blocks of ", QB);
  check(codes, "codes", torch::kUInt8, 2 * n, codes);
  check(exps, "exps", torch::kUInt8, 2 * (n / QB), codes);
  const c10::DeviceGuard guard(codes.device());
  auto m = torch::empty({n}, codes.options().dtype(torch::kBFloat16));
  auto v = torch::empty_like(m);
  if (n == 0) return {m, v};
  const long quads = n / 4;
  const int grid = (int)std::min<long>((quads + BLOCK - 1) / BLOCK, 4096L);
  moments_kernel<<<grid, BLOCK, 0, cur_stream()>>>(
      reinterpret_cast<const uint2*>(codes.data_ptr()),
      reinterpret_cast<const uchar2*>(exps.data_ptr()),
      reinterpret_cast<bf16x4*>(m.data_ptr()),
      reinterpret_cast<bf16x4*>(v.data_ptr()), quads);
  return {m, v};
}

}  // namespace eg
