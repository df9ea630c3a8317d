// Dropout from a counter-based generator: y = keep ? x / (1 - p) : 0, where keep is
// a function of (seed, place), so that the backward pass makes the same mask again
// and nobody stores it.
//
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011): key = the seed's 64 bits, counter = the index of a group of eight
// elements.  Its four words are eight numbers of 16 bits; an element stays if its
// number is at least ``drop`` = p in 65536ths, and is multiplied by
// 65536 / (65536 - drop), so that the expectation is x whatever p was rounded to.
//
// What bounds it: memory (8192 x 14336 bf16, forward and backward, 175 us, 5.4 TB/s; 8192 x
// 4096 53 us).  Of a group 20 products of 32 x 32 bits, at 16 cycles each, make its numbers; 32 bits
// for each element would take twice as many, about the time that memory takes.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "common.h"

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

DEV_INLINE u32x4_t philox(uint64_t at, uint32_t k0, uint32_t k1) {
  uint32_t c0 = (uint32_t)at, c1 = (uint32_t)(at >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4_t{c0, c1, c2, c3};
}

DEV_INLINE uint32_t bits_of(const u32x4_t& r, int j) {
  return j % 2 ? r[j / 2] >> 16 : r[j / 2] & 0xffffu;
}

template <typename T>
DEV_INLINE T kept(T x, bool keep, float scale) {
  return keep ? (T)((float)x * scale) : (T)0.f;
}

template <typename T>
struct alignas(16) Eight {
  T v[8];
};

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(
    T* __restrict__ out, const T* __restrict__ x, const int64_t* __restrict__ seed,
    long n, uint32_t drop, float scale) {
  const uint64_t key = (uint64_t)seed[0];
  const long whole = n / 8, stride = (long)gridDim.x * 256;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i * 8 < n; i += stride) {
    const u32x4_t r = philox((uint64_t)i, (uint32_t)key, (uint32_t)(key >> 32));
    if (i < whole) {
      Eight<T> w = reinterpret_cast<const Eight<T>*>(x)[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) w.v[j] = kept(w.v[j], bits_of(r, j) >= drop, scale);
      reinterpret_cast<Eight<T>*>(out)[i] = w;
    } else {
      for (int j = 0; j < (int)(n - whole * 8); ++j)
        out[i * 8 + j] = kept(x[i * 8 + j], bits_of(r, j) >= drop, scale);
    }
  }
}

static torch::Tensor dropout(torch::Tensor x, int64_t drop, const torch::Tensor& seed) {
  TORCH_CHECK(x.is_cuda(), "dropout: x on the GPU");
  x = x.contiguous();
  if ((uintptr_t)x.data_ptr() & 15) x = x.clone();
  TORCH_CHECK(seed.device() == x.device() && seed.scalar_type() == torch::kInt64 &&
                  seed.numel() == 1,
              "dropout: seed (1) int64 on x's device");
  TORCH_CHECK(drop >= 0 && drop <= 65536, "dropout: drop in 0 .. 65536");
  const c10::DeviceGuard guard(x.device());
  auto out = torch::empty_like(x);
  const long n = x.numel();
  if (n == 0) return out;
  const float scale = drop < 65536 ? 65536.f / (float)(65536 - drop) : 0.f;
  const unsigned blocks = (unsigned)std::min<long>((n + 2047) / 2048, MAX_RESIDENT_BLOCKS);
  auto go = [&](auto t) {
    using T = decltype(t);
    dropout_kernel<T><<<dim3(blocks), dim3(256), 0, at::hip::getCurrentHIPStream()>>>(
        (T*)out.data_ptr(), (const T*)x.data_ptr(), seed.data_ptr<int64_t>(), n,
        (uint32_t)drop, scale);
  };
  if (x.scalar_type() == torch::kBFloat16) go(__bf16{});
  else if (x.scalar_type() == torch::kFloat16) go(_Float16{});
  else if (x.scalar_type() == torch::kFloat32) go(float{});
  else TORCH_CHECK(false, "dropout: dtype must be bf16, fp16 or fp32");
  HIP_CHECK_KERNEL();
  return out;
}

// The way back makes the mask again, so that it is the same function of dy.  (In C++: a
// small call and its gradient take 46 us, through Python's autograd functions 75; the
// kernels take 5.)
struct Dropout : torch::autograd::Function<Dropout> {
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx,
                               const torch::Tensor& x, int64_t drop,
                               const torch::Tensor& seed) {
    ctx->save_for_backward({seed});
    ctx->saved_data["drop"] = drop;
    return dropout(x, drop, seed);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list dy) {
    const auto seed = ctx->get_saved_variables()[0];
    return {Dropout::apply(dy[0], ctx->saved_data["drop"].toInt(), seed), {}, {}};
  }
};

torch::Tensor dropout_train(const torch::Tensor& x, int64_t drop,
                            const torch::Tensor& seed) {
  return Dropout::apply(x, drop, seed);
}
