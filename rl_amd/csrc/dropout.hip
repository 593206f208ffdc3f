// Dropout from a counter-based generator: the mask is a function of (seed, offset, element
// number), so the backward forms it again and nothing is stored.
//
// Elements 8 q .. 8 q + 7 of a tensor take the eight 16-bit pieces (low pieces first) of one
// Philox4x32-10 block (Salmon, Moraes, Dror and Shaw, SC 2011) with the 64-bit seed as key and
// (q, offset) as counter; element i is kept where its piece u >= T, T = floor(p * 65536 + 1/2),
// and multiplied by 65536 / (65536 - T).  16 bits per element place p within 2^-17 of what was
// asked; the factor belongs to the p that is drawn, so the expectation is exact.  With 32 bits
// per element the generator's multiplications alone would take as long as the memory traffic.
//
// Bound by memory, each element read and written once: [16384, 4096] bf16 42 us, 6.4 TB/s.

#include "philox.h"

namespace mirl {
namespace {

constexpr int kV = 8;
constexpr int kThreads = 256;

template <class E>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const typename E::raw* x, int64_t n,
                                                           DropoutArgs D, typename E::raw* y) {
  const uint64_t seed = D.seed_of();
  for (int64_t q = (int64_t)blockIdx.x * kThreads + threadIdx.x; q * kV < n; q += (int64_t)gridDim.x * kThreads) {
    const int64_t i = q * kV;
    if (i + kV <= n) {
      // any alignment of an element, each used once
      using piece = typename Piece<alignof(typename E::raw)>::type;
      constexpr int kP = kV / E::kVec;
      vu4 q4[kP];
#pragma unroll
      for (int k = 0; k < kP; ++k) q4[k] = __builtin_nontemporal_load(reinterpret_cast<const piece*>(x + i) + k);
      const uint32_t keep = dropout_keep8(seed, D.offset, (uint64_t)q, D.threshold);
#pragma unroll
      for (int k = 0; k < kP; ++k) {
        float v[E::kVec];
        E::unpack(q4[k], v);
#pragma unroll
        for (int e = 0; e < E::kVec; ++e) v[e] = (keep >> (k * E::kVec + e)) & 1u ? v[e] * D.scale : 0.f;
        __builtin_nontemporal_store((piece)E::pack(v), reinterpret_cast<piece*>(y + i) + k);
      }
    } else {
      const uint32_t keep = dropout_keep8(seed, D.offset, (uint64_t)q, D.threshold);
      for (int e = 0; i + e < n; ++e)
        y[i + e] = E::from_float((keep >> e) & 1u ? E::load(x + i + e) * D.scale : 0.f);
    }
  }
}

}  // namespace
}  // namespace mirl

using namespace mirl;

extern "C" int mirl_dropout(const void* x, int dtype, int64_t n, double p, int64_t seed, const int64_t* seed_dev,
                            int64_t offset, void* y, void* stream) {
  clear_error();
  MIRL_REQUIRE(n >= 0, "invalid element count %lld", (long long)n);
  MIRL_REQUIRE(p >= 0.0 && p <= 1.0, "dropout probability %g is outside [0, 1]", p);
  MIRL_REQUIRE(dtype == MIRL_DTYPE_F32 || dtype == MIRL_DTYPE_BF16 || dtype == MIRL_DTYPE_F16,
               "dropout takes fp32, bf16 or fp16 (dtype code %d)", dtype);
  if (n == 0) return MIRL_OK;
  MIRL_REQUIRE(x && y, "null pointer argument");
  const DropoutArgs D = dropout_args(p, seed, seed_dev, offset);
  // a launch holds fewer than 2^32 threads; the workgroups stride over more elements
  const int64_t blocks = (n + kThreads * kV - 1) / (kThreads * kV), most = int64_t(1) << 20;
  const int64_t grid = blocks < most ? blocks : most;
  auto launch = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL(dropout_kernel<E>, dim3((unsigned)grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<const typename E::raw*>(x), n, D, static_cast<typename E::raw*>(y));
  };
  if (dtype == MIRL_DTYPE_F32)
    launch(F32{});
  else if (dtype == MIRL_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return check_launch("mirl_dropout");
}
