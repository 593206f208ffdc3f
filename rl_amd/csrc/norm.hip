// Root-mean-square norm of the residual stream, with the residual's addition, for
// training (with its backward) and for scoring in 8 bits.
//
//   h    = EH(x + res)                       the stream as it is stored (h = x without res)
//   n    = h * rstd,  rstd = 1 / sqrt(mean(h^2) + eps)
//   y    = EX(n * w)                         or, in 8 bits, e4m3(y * (1 / s)) with s = max|y| / 448,
//                                            or int8 of it, to the nearest, with s = max|y| / 127
//   dh   = rstd * (w dy - n * mean(w dy n)) + dh_out,   dw = sum over rows of dy * n
//
// Every sum is fp32; y, h, dx, dres and dw are rounded once, to the types of the tensors that
// hold them.  n is formed from the rounded h, so that the backward, which reads the stored h,
// differentiates what the forward computed.
//
// Bound by memory: the row stays in registers between its two uses (its sum of squares and
// its output; the largest magnitude as well in 8 bits), so each input is read once and each
// output written once.  Rows of up to 16384 elements are held by one wave (H <= 1024, four
// rows a workgroup) or by a workgroup; longer ones are read again instead.
//
// Measured on [16384, 4096] bf16: forward 94 us (537 MB, 5.7 TB/s), with the 8-bit output 88
// (470 MB, 5.3), backward 102 and 6 for dw's sum (537 MB, 5.3); the library's copy of 4 GiB
// moves 4.75 TB/s, dropout.hip 6.4.  Four waves a row: with one wave (64 values a lane) 171
// and 245 us, with eight 93 and 105, but 107 with the 8-bit output.  Plain stores or loads
// instead of nontemporal ones: the same within 1%.  What is left is the pause of a workgroup
// between its loads and its stores; the next row's loads ahead of them (141 registers) took
// the backward from 104 to 118 us.

#include "common.h"

namespace mirl {
namespace {

constexpr int kV = 8;  // elements a lane handles together

// Eight elements at p, which is aligned to one element only (odd hidden sizes put rows
// anywhere): one or two 16-byte pieces, which the hardware takes unaligned.  Nontemporal:
// each is used once.
template <class E>
__device__ __forceinline__ void load8(const typename E::raw* p, float (&v)[kV]) {
#pragma unroll
  for (int i = 0; i < kV / E::kVec; ++i) {
    using piece = typename Piece<alignof(typename E::raw)>::type;
    const vu4 q = __builtin_nontemporal_load(reinterpret_cast<const piece*>(p) + i);
    float w[E::kVec];
    E::unpack(q, w);
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) v[i * E::kVec + e] = w[e];
  }
}
template <class E>
__device__ __forceinline__ void store8(typename E::raw* p, const float (&v)[kV]) {
#pragma unroll
  for (int i = 0; i < kV / E::kVec; ++i) {
    using piece = typename Piece<alignof(typename E::raw)>::type;
    float w[E::kVec];
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) w[e] = v[i * E::kVec + e];
    __builtin_nontemporal_store((piece)E::pack(w), reinterpret_cast<piece*>(p) + i);
  }
}
// Elements c .. c + 7 of a row of H, zeros past its end.
template <class E>
__device__ __forceinline__ void load8_to(const typename E::raw* row, int64_t c, int64_t H, float (&v)[kV]) {
  if (c + kV <= H) {
    load8<E>(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = c + e < H ? E::load(row + c + e) : 0.f;
  }
}
template <class E>
__device__ __forceinline__ void store8_to(typename E::raw* row, int64_t c, int64_t H, const float (&v)[kV]) {
  if (c + kV <= H) {
    store8<E>(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e)
      if (c + e < H) row[c + e] = E::from_float(v[e]);
  }
}

// The norm's weight, of the rows' type or fp32.
struct Weight {
  const void* p;
  int f32;
};
template <class EX>
__device__ __forceinline__ void load_weight(const Weight& w, int64_t c, int64_t H, float (&v)[kV]) {
  if (std::is_same<EX, F32>::value || w.f32)
    load8_to<F32>(static_cast<const float*>(w.p), c, H, v);
  else
    load8_to<EX>(static_cast<const typename EX::raw*>(w.p), c, H, v);
}

// e4m3 of eight values (round to nearest even), as 8 bytes.
__device__ __forceinline__ uint2 pack_e4m3(const float (&v)[kV]) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return uint2{(uint32_t)lo, (uint32_t)hi};
}
// Eight values of at most 127 to the nearest whole number (ties to the even one; NaN becomes 0).
__device__ __forceinline__ uint2 pack_int8(const float (&v)[kV]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = (uint32_t)(int)rintf(v[4 * i + e]);
    w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u),
                                 0x05040100u);
  }
  return uint2{w[0], w[1]};
}
struct __attribute__((packed, aligned(1))) Bytes8 {
  uint32_t lo, hi;
};
// What the rows become: the type of the input, or 8 bits with a scale.
enum Out { kSame = 0, kE4m3 = 1, kInt8 = 2 };
template <int OUT>
__device__ __forceinline__ void store_8bit(uint8_t* row, int64_t c, int64_t H, const float (&v)[kV]) {
  const uint2 q = OUT == kInt8 ? pack_int8(v) : pack_e4m3(v);
  if (c + kV <= H) {
    *reinterpret_cast<Bytes8*>(row + c) = Bytes8{q.x, q.y};
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e)
      if (c + e < H) row[c + e] = (uint8_t)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
  }
}

constexpr float kE4m3Max = 448.f, kInt8Max = 127.f;
constexpr uint32_t kAbs = 0x7fffffffu;
// The scale of a row whose largest magnitude has these bits: amax / 448 (int8: 127), not below the
// smallest normal number (so that its reciprocal is finite), 1 for a row of zeros.  The
// magnitudes are compared as integers: a NaN is then the largest and makes the row NaN.
template <int OUT>
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits);
  if (amax_bits == 0) return 1.f;
  const float s = amax / (OUT == kInt8 ? kInt8Max : kE4m3Max);
  return s < 0x1p-126f ? 0x1p-126f : s;
}

// Sums (or integer maxima) over the NW waves that share a row; s holds one slot per wave and
// row.  Two barriers, so that the slots can be used again.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, off, kWave);
    v = o > v ? o : v;
  }
  return v;
}
template <int NW>
__device__ __forceinline__ float row_sum(float v, float* s) {
  v = wave_sum(v);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += s[i];
  }
  return v;
}
template <int NW>
__device__ __forceinline__ uint32_t row_umax(uint32_t v, float* s) {
  v = wave_umax(v);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[wave] = __uint_as_float(v);
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const uint32_t o = __float_as_uint(s[i]);
      v = o > v ? o : v;
    }
  }
  return v;
}

struct NormFwd {
  const void* x;
  const void* res;  // or null
  int64_t ldx, ldr;
  Weight w;
  int64_t R, H;
  float eps;
  void* h;          // [R, H] of EH (null without res: the stream is x)
  void* y;          // [R, H] of EX, or e4m3 bytes
  float* scale;     // [R], 8-bit output only
  float* rstd;      // [R] or null
};

// Rows of up to 64 * NW * kV * NV elements, in registers: NW waves a row (4 / NW rows a
// workgroup where NW < 4).
template <class EX, class EH, int NW, int NV, int OUT>
__global__ __launch_bounds__(NW < 4 ? 256 : 64 * NW) void norm_fwd_kernel(NormFwd P) {
  constexpr int kRowsPerWg = NW < 4 ? 4 / NW : 1;
  static_assert(NW == 1 || NW >= 4, "one wave or the workgroup per row");
  __shared__ float s[NW];
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
  // (whole waves leave the loop where NW == 1, which has no barrier)
  for (int64_t r = (int64_t)blockIdx.x * kRowsPerWg + (NW == 1 ? threadIdx.x >> 6 : 0); r < P.R;
       r += (int64_t)gridDim.x * kRowsPerWg) {
    const typename EX::raw* xr = static_cast<const typename EX::raw*>(P.x) + r * P.ldx;
    float h[NV][kV];
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) load8_to<EX>(xr, (int64_t)(k * NW * 64 + t) * kV, P.H, h[k]);
    if (P.res != nullptr) {
      const typename EH::raw* rr = static_cast<const typename EH::raw*>(P.res) + r * P.ldr;
      typename EH::raw* hr = static_cast<typename EH::raw*>(P.h) + r * P.H;
      float q[NV][kV];
#pragma unroll
      for (int k = 0; k < NV; ++k) load8_to<EH>(rr, (int64_t)(k * NW * 64 + t) * kV, P.H, q[k]);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int e = 0; e < kV; ++e) h[k][e] = round_trip<EH>(h[k][e] + q[k][e]);
        const int64_t c = (int64_t)(k * NW * 64 + t) * kV;
        if (c < P.H) store8_to<EH>(hr, c, P.H, h[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < kV; ++e) sq = fmaf(h[k][e], h[k][e], sq);
    sq = row_sum<NW>(sq, s);
    const float rstd = 1.f / sqrtf(sq / (float)P.H + P.eps);
    if (P.rstd != nullptr && t == 0) P.rstd[r] = rstd;
    uint32_t amax = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = (int64_t)(k * NW * 64 + t) * kV;
      if (c >= P.H) continue;
      float w[kV];
      load_weight<EX>(P.w, c, P.H, w);
#pragma unroll
      for (int e = 0; e < kV; ++e) h[k][e] = (h[k][e] * rstd) * w[e];
      if constexpr (OUT != kSame) {
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          // past the row's end h is 0 and w is 0; a NaN rstd must not reach those
          const uint32_t a = c + e < P.H ? __float_as_uint(h[k][e]) & kAbs : 0u;
          amax = a > amax ? a : amax;
        }
      } else {
        store8_to<EX>(static_cast<typename EX::raw*>(P.y) + r * P.H, c, P.H, h[k]);
      }
    }
    if constexpr (OUT != kSame) {
      amax = row_umax<NW>(amax, s);
      const float sc = row_scale<OUT>(amax), inv = 1.f / sc;
      if (t == 0) P.scale[r] = sc;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int64_t c = (int64_t)(k * NW * 64 + t) * kV;
        if (c >= P.H) continue;
#pragma unroll
        for (int e = 0; e < kV; ++e) h[k][e] *= inv;
        store_8bit<OUT>(static_cast<uint8_t*>(P.y) + r * P.H, c, P.H, h[k]);
      }
    }
  }
}

// Longer rows: a workgroup of 16 waves reads the row once for the sum of squares (and writes
// h), again for the output (from h, which this workgroup wrote: each thread reads what it
// wrote itself), and for an 8-bit output once more.
constexpr int kLongThreads = 1024;
template <class EX, class EH, int OUT>
__global__ __launch_bounds__(kLongThreads) void norm_fwd_long_kernel(NormFwd P) {
  constexpr int NW = kLongThreads / kWave;
  __shared__ float s[NW];
  for (int64_t r = blockIdx.x; r < P.R; r += gridDim.x) {
    const typename EX::raw* xr = static_cast<const typename EX::raw*>(P.x) + r * P.ldx;
    const typename EH::raw* rr = static_cast<const typename EH::raw*>(P.res) + (P.res ? r * P.ldr : 0);
    typename EH::raw* hr = static_cast<typename EH::raw*>(P.h) + (P.res ? r * P.H : 0);
    float sq = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * kV; c < P.H; c += kLongThreads * kV) {
      float h[kV];
      load8_to<EX>(xr, c, P.H, h);
      if (P.res != nullptr) {
        float q[kV];
        load8_to<EH>(rr, c, P.H, q);
#pragma unroll
        for (int e = 0; e < kV; ++e) h[e] = round_trip<EH>(h[e] + q[e]);
        store8_to<EH>(hr, c, P.H, h);
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) sq = fmaf(h[e], h[e], sq);
    }
    sq = row_sum<NW>(sq, s);
    const float rstd = 1.f / sqrtf(sq / (float)P.H + P.eps);
    if (P.rstd != nullptr && threadIdx.x == 0) P.rstd[r] = rstd;
    auto value = [&](int64_t c, float (&y)[kV]) {
      if (P.res != nullptr)
        load8_to<EH>(hr, c, P.H, y);
      else
        load8_to<EX>(xr, c, P.H, y);
      float w[kV];
      load_weight<EX>(P.w, c, P.H, w);
#pragma unroll
      for (int e = 0; e < kV; ++e) y[e] = (y[e] * rstd) * w[e];
    };
    float inv = 1.f;
    if constexpr (OUT != kSame) {
      uint32_t amax = 0;
      for (int64_t c = (int64_t)threadIdx.x * kV; c < P.H; c += kLongThreads * kV) {
        float y[kV];
        value(c, y);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          const uint32_t a = c + e < P.H ? __float_as_uint(y[e]) & kAbs : 0u;
          amax = a > amax ? a : amax;
        }
      }
      amax = row_umax<NW>(amax, s);
      const float sc = row_scale<OUT>(amax);
      inv = 1.f / sc;
      if (threadIdx.x == 0) P.scale[r] = sc;
    }
    for (int64_t c = (int64_t)threadIdx.x * kV; c < P.H; c += kLongThreads * kV) {
      float y[kV];
      value(c, y);
      if constexpr (OUT != kSame) {
#pragma unroll
        for (int e = 0; e < kV; ++e) y[e] *= inv;
        store_8bit<OUT>(static_cast<uint8_t*>(P.y) + r * P.H, c, P.H, y);
      } else {
        store8_to<EX>(static_cast<typename EX::raw*>(P.y) + r * P.H, c, P.H, y);
      }
    }
  }
}

// Rows in 8 bits without a norm (an output weight's): one workgroup per row, read twice (the
// second time from the cache for rows of ordinary length).  [151936, 4096] bf16 499 us, once per
// set of weights: 3.7 TB/s with each element read and written once, 6.4 being what streams reach;
// a workgroup's second pass waits for the row's maximum.
template <class EX, int OUT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const typename EX::raw* __restrict__ x, int64_t ldx,
                                                            int64_t R, int64_t H, uint8_t* __restrict__ y,
                                                            float* __restrict__ scale) {
  __shared__ float s[4];
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const typename EX::raw* xr = x + r * ldx;
    uint32_t amax = 0;
    for (int64_t c = (int64_t)threadIdx.x * kV; c < H; c += 256 * kV) {
      float v[kV];
      load8_to<EX>(xr, c, H, v);
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        const uint32_t a = __float_as_uint(v[e]) & kAbs;
        amax = a > amax ? a : amax;
      }
    }
    amax = row_umax<4>(amax, s);
    const float sc = row_scale<OUT>(amax), inv = 1.f / sc;
    if (threadIdx.x == 0) scale[r] = sc;
    for (int64_t c = (int64_t)threadIdx.x * kV; c < H; c += 256 * kV) {
      float v[kV];
      load8_to<EX>(xr, c, H, v);
#pragma unroll
      for (int e = 0; e < kV; ++e) v[e] *= inv;
      store_8bit<OUT>(y + r * H, c, H, v);
    }
  }
}

struct NormBwd {
  const void* dy;      // [R, H] of EX, row stride lddy
  int64_t lddy;
  const void* dh_out;  // [R, H] of EH (the gradient of the stream), row stride ldd, or null
  int64_t ldd;
  const void* h;       // [R, H] of EH, row stride ldh
  int64_t ldh;
  const float* rstd;
  Weight w;
  int64_t R, H;
  void* dx;            // [R, H] of EX, or null
  void* dres;          // [R, H] of EH, or null
  float* dw_part;      // [groups, H] or null
  int64_t groups;      // rows group, group + groups, ... belong to one partial sum of dw
  void* dw;            // [H] of the weight's type, written by the workgroups from dw_first on, or null
  int64_t dw_first;
};

// dw of 16 columns by one workgroup that reads them again: for rows few enough to lie in the
// caches, beside the workgroups that form dh, in place of partial sums and a second launch.  A
// lane's rows go into eight sums and the lanes' sums into four: at most R / 128 + 10 additions in
// sequence with 16 lanes a column, 22 with 64.
template <class EX, class EH>
__device__ __forceinline__ void dw_columns(const NormBwd& P, int64_t block, float (*s)[17]) {
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, lanes = blockDim.x >> 4;
  const int64_t c = block * 16 + cl;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (c < P.H) {
    const typename EX::raw* d = static_cast<const typename EX::raw*>(P.dy) + rl * P.lddy + c;
    const typename EH::raw* h = static_cast<const typename EH::raw*>(P.h) + rl * P.ldh + c;
    const int64_t sd = lanes * P.lddy, sh = lanes * P.ldh;
    // n of the lane's rows from r on, the first `have` of them there (the others are read as the first)
    auto rows = [&](auto n_c, int64_t r, int64_t have) __attribute__((always_inline)) {
      constexpr int N = decltype(n_c)::value;
      float dv[N], hv[N], rs[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t k = i < have ? i : 0;
        dv[i] = EX::load(d + k * sd);
        hv[i] = EH::load(h + k * sh);
        rs[i] = P.rstd[r + k * lanes];
      }
      __builtin_amdgcn_sched_barrier(0);  // all loads in flight before the first sum waits
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = i < have ? fmaf(dv[i], hv[i] * rs[i], v[i]) : v[i];
    };
    int64_t r = rl;
    for (; r + 7 * lanes < P.R; r += 8 * lanes) {
      rows(std::integral_constant<int, 8>{}, r, 8);
      d += 8 * sd;
      h += 8 * sh;
    }
    if (r + lanes < P.R)
      rows(std::integral_constant<int, 7>{}, r, (P.R - r + lanes - 1) / lanes);
    else if (r < P.R)
      rows(std::integral_constant<int, 1>{}, r, 1);
  }
  s[rl][cl] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  __syncthreads();
  if (threadIdx.x < 16 && c < P.H) {
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < lanes; i += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] += s[i + e][cl];
    const float sum = (t[0] + t[1]) + (t[2] + t[3]);
    if (std::is_same<EX, F32>::value || P.w.f32)
      static_cast<float*>(P.dw)[c] = sum;
    else
      static_cast<typename EX::raw*>(P.dw)[c] = EX::from_float(sum);
  }
}

// One wave (NW == 1) or workgroup per group of rows; the row's two operands stay in registers
// between the reduction and the output, and the columns' sums of dy * n across the group.
template <class EX, class EH, int NW, int NV>
__global__ __launch_bounds__(NW < 4 ? 256 : 64 * NW) void norm_bwd_kernel(NormBwd P) {
  constexpr int kRowsPerWg = NW < 4 ? 4 / NW : 1;
  __shared__ float s[NW];
  __shared__ float s_dw[(NW < 4 ? 256 : 64 * NW) / 16][17];
  if (P.dw != nullptr && (int64_t)blockIdx.x >= P.dw_first) {
    dw_columns<EX, EH>(P, blockIdx.x - P.dw_first, s_dw);
    return;
  }
  const int64_t g = (int64_t)blockIdx.x * kRowsPerWg + (NW == 1 ? threadIdx.x >> 6 : 0);
  if (g >= P.groups) return;
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
  float w[NV][kV], dw[NV][kV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_weight<EX>(P.w, (int64_t)(k * NW * 64 + t) * kV, P.H, w[k]);
#pragma unroll
    for (int e = 0; e < kV; ++e) dw[k][e] = 0.f;
  }
  const float inv_h = 1.f / (float)P.H;
  for (int64_t r = g; r < P.R; r += P.groups) {
    const typename EX::raw* dyr = static_cast<const typename EX::raw*>(P.dy) + r * P.lddy;
    const typename EH::raw* hr = static_cast<const typename EH::raw*>(P.h) + r * P.ldh;
    float n[NV][kV], d[NV][kV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = (int64_t)(k * NW * 64 + t) * kV;
      load8_to<EX>(dyr, c, P.H, d[k]);
      load8_to<EH>(hr, c, P.H, n[k]);
    }
    const float rstd = P.rstd[r];
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        n[k][e] *= rstd;
        dw[k][e] = fmaf(d[k][e], n[k][e], dw[k][e]);
        d[k][e] *= w[k][e];
        dot = fmaf(d[k][e], n[k][e], dot);
      }
    dot = row_sum<NW>(dot, s) * inv_h;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = (int64_t)(k * NW * 64 + t) * kV;
      if (c >= P.H) continue;
      float o[kV];
      if (P.dh_out != nullptr) {
        load8_to<EH>(static_cast<const typename EH::raw*>(P.dh_out) + r * P.ldd, c, P.H, o);
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) o[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) o[e] = fmaf(rstd, fmaf(-n[k][e], dot, d[k][e]), o[e]);
      if (P.dx != nullptr) store8_to<EX>(static_cast<typename EX::raw*>(P.dx) + r * P.H, c, P.H, o);
      if (P.dres != nullptr) store8_to<EH>(static_cast<typename EH::raw*>(P.dres) + r * P.H, c, P.H, o);
    }
  }
  if (P.dw_part != nullptr) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = (int64_t)(k * NW * 64 + t) * kV;
      if (c < P.H) store8_to<F32>(P.dw_part + g * P.H, c, P.H, dw[k]);
    }
  }
}

// Longer rows: read once for the reduction and once for the output.  dw by one more kernel.
template <class EX, class EH>
__global__ __launch_bounds__(kLongThreads) void norm_bwd_long_kernel(NormBwd P) {
  constexpr int NW = kLongThreads / kWave;
  __shared__ float s[NW];
  for (int64_t r = blockIdx.x; r < P.R; r += gridDim.x) {
    const typename EX::raw* dyr = static_cast<const typename EX::raw*>(P.dy) + r * P.lddy;
    const typename EH::raw* hr = static_cast<const typename EH::raw*>(P.h) + r * P.ldh;
    const float rstd = P.rstd[r];
    auto operands = [&](int64_t c, float (&n)[kV], float (&d)[kV]) {
      float w[kV];
      load8_to<EX>(dyr, c, P.H, d);
      load8_to<EH>(hr, c, P.H, n);
      load_weight<EX>(P.w, c, P.H, w);
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        n[e] *= rstd;
        d[e] *= w[e];
      }
    };
    float dot = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * kV; c < P.H; c += kLongThreads * kV) {
      float n[kV], d[kV];
      operands(c, n, d);
#pragma unroll
      for (int e = 0; e < kV; ++e) dot = fmaf(d[e], n[e], dot);
    }
    dot = row_sum<NW>(dot, s) / (float)P.H;
    for (int64_t c = (int64_t)threadIdx.x * kV; c < P.H; c += kLongThreads * kV) {
      float n[kV], d[kV], o[kV];
      operands(c, n, d);
      if (P.dh_out != nullptr) {
        load8_to<EH>(static_cast<const typename EH::raw*>(P.dh_out) + r * P.ldd, c, P.H, o);
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) o[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) o[e] = fmaf(rstd, fmaf(-n[e], dot, d[e]), o[e]);
      if (P.dx != nullptr) store8_to<EX>(static_cast<typename EX::raw*>(P.dx) + r * P.H, c, P.H, o);
      if (P.dres != nullptr) store8_to<EH>(static_cast<typename EH::raw*>(P.dres) + r * P.H, c, P.H, o);
    }
  }
}
// dw's partial sums of longer rows: workgroup (column block, group), eight columns a thread.
template <class EX, class EH>
__global__ __launch_bounds__(256) void norm_dw_long_kernel(NormBwd P) {
  const int64_t n_cb = (P.H + 256 * kV - 1) / (256 * kV);
  const int64_t g = blockIdx.x / n_cb, c = ((blockIdx.x - g * n_cb) * 256 + threadIdx.x) * kV;
  if (c >= P.H) return;
  float dw[kV];
#pragma unroll
  for (int e = 0; e < kV; ++e) dw[e] = 0.f;
  for (int64_t r = g; r < P.R; r += P.groups) {
    float d[kV], n[kV];
    load8_to<EX>(static_cast<const typename EX::raw*>(P.dy) + r * P.lddy, c, P.H, d);
    load8_to<EH>(static_cast<const typename EH::raw*>(P.h) + r * P.ldh, c, P.H, n);
    const float rstd = P.rstd[r];
#pragma unroll
    for (int e = 0; e < kV; ++e) dw[e] = fmaf(d[e], n[e] * rstd, dw[e]);
  }
  store8_to<F32>(P.dw_part + g * P.H, c, P.H, dw);
}

// dw[c] = EW(sum over groups of part[g][c]), in an order that depends on the sizes only: 32
// columns a workgroup, 32 lanes of groups each.
template <class EW>
__global__ __launch_bounds__(1024) void norm_dw_sum_kernel(const float* __restrict__ part, int64_t groups, int64_t H,
                                                           typename EW::raw* __restrict__ dw) {
  __shared__ float s[32][33];
  const int cl = threadIdx.x & 31, gl = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + cl;
  float v = 0.f;
  if (c < H) {
#pragma unroll 8
    for (int64_t g = gl; g < groups; g += 32) v += part[g * H + c];
  }
  s[gl][cl] = v;
  __syncthreads();
  // thread (gl, cl) now holds column gl, group lane cl
  v = s[cl][gl];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  const int64_t oc = (int64_t)blockIdx.x * 32 + gl;
  if (cl == 0 && oc < H) dw[oc] = EW::from_float(v);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// f(EX, EH) for the supported pairs of row and stream types: the stream has the rows' type or
// fp32.
template <class F>
int with_types(int x_dtype, int h_dtype, F&& f) {
  if (x_dtype == MIRL_DTYPE_F32 && h_dtype == MIRL_DTYPE_F32) return f(F32{}, F32{});
  if (x_dtype == MIRL_DTYPE_BF16 && h_dtype == MIRL_DTYPE_BF16) return f(BF16{}, BF16{});
  if (x_dtype == MIRL_DTYPE_BF16 && h_dtype == MIRL_DTYPE_F32) return f(BF16{}, F32{});
  if (x_dtype == MIRL_DTYPE_F16 && h_dtype == MIRL_DTYPE_F16) return f(F16{}, F16{});
  if (x_dtype == MIRL_DTYPE_F16 && h_dtype == MIRL_DTYPE_F32) return f(F16{}, F32{});
  set_error("the rows are fp32, bf16 or fp16 and the residual of their type or fp32 (dtype codes %d and %d)",
            x_dtype, h_dtype);
  return MIRL_ERR_INVALID_ARGUMENT;
}
// f(NW, NV) for the layout of rows of H elements that registers hold, the longer ones' f(0, 0).
template <int A, int B>
struct Layout {
  static constexpr int kNW = A, kNV = B;
};
template <class F>
int with_layout(int64_t H, F&& f) {
  if (H <= 512) return f(Layout<1, 1>{});
  if (H <= 1024) return f(Layout<1, 2>{});
  if (H <= 2048) return f(Layout<4, 1>{});
  if (H <= 4096) return f(Layout<4, 2>{});
  if (H <= 8192) return f(Layout<8, 2>{});
  if (H <= 16384) return f(Layout<16, 2>{});
  return f(Layout<0, 0>{});
}

int check_weight(int x_dtype, int w_dtype) {
  MIRL_REQUIRE(w_dtype == x_dtype || w_dtype == MIRL_DTYPE_F32,
               "the weight has the rows' type or fp32 (dtype codes %d and %d)", w_dtype, x_dtype);
  return MIRL_OK;
}
constexpr int64_t kMaxSide = int64_t(1) << 31, kMaxWidth = int64_t(1) << 24;
// Batches whose dw is formed from a second read, in the same launch: of few elements (forward and
// backward of [257, 3, 1021] fp32 with autograd around them: 114 us with partial sums and a launch more,
// 106 so) in few rows, which a column's 16 lanes share.  Kernels alone, second read against partial sums, us:
// bf16 [771, 1021] 5.7 and 12.4, [2048, 512] 8.2 and 10.5, [2048, 64] 7.8 and 9.1, [2048, 17] 9.1 and 9.5,
// [4096, 64] 13.3 and 11.2, [16384, 17] 57 and 28, [60000, 17] 303 and 83.
constexpr int64_t kFewElems = int64_t(1) << 20, kFewRows = 2048;
bool few_rows(int64_t R, int64_t H) { return H <= 16384 && R <= kFewRows && R * H <= kFewElems; }
// Partial sums of dw: four workgroups per CU (eight: 108 and 11 us of [16384, 4096] against 104
// and 6; three: 6% more).
constexpr int64_t kMaxGroups = 1024;
// Workgroups of a launch over rows (a launch holds fewer than 2^32 threads); they stride over more rows.
constexpr int64_t kMaxGrid = int64_t(1) << 20;
unsigned row_grid(int64_t n) { return (unsigned)(n < kMaxGrid ? n : kMaxGrid); }

}  // namespace
}  // namespace mirl

using namespace mirl;

namespace mirl {
namespace {
int norm_fwd(int out, const void* x, int x_dtype, int64_t ldx, const void* residual, int res_dtype, int64_t ldr,
             const void* weight, int w_dtype, int64_t R, int64_t H, double eps, void* h, void* y, float* y_scale,
             float* rstd, void* stream) {
  clear_error();
  MIRL_REQUIRE(R >= 0 && H > 0 && R < kMaxSide && H < kMaxWidth, "invalid shape R=%lld H=%lld", (long long)R, (long long)H);
  MIRL_REQUIRE(eps >= 0, "eps %g is negative", eps);
  const int h_dtype = residual != nullptr ? res_dtype : x_dtype;
  if (int e = check_weight(x_dtype, w_dtype)) return e;
  return with_types(x_dtype, h_dtype, [&](auto ex, auto eh) -> int {
    using EX = decltype(ex);
    using EH = decltype(eh);
    if (R == 0) return MIRL_OK;
    MIRL_REQUIRE(x && weight && y && (residual == nullptr || h != nullptr), "null pointer argument");
    MIRL_REQUIRE((R == 1 || ldx >= H) && (residual == nullptr || R == 1 || ldr >= H),
                 "row strides (%lld, %lld) are below H=%lld", (long long)ldx, (long long)ldr, (long long)H);
    const NormFwd P{x, residual, ldx, ldr, Weight{weight, w_dtype == MIRL_DTYPE_F32}, R, H, (float)eps, h, y, y_scale, rstd};
    hipStream_t st = static_cast<hipStream_t>(stream);
    return with_layout(H, [&](auto layout) -> int {
      using L = decltype(layout);
      auto go = [&](auto out_c) {
        constexpr int OUT = decltype(out_c)::value;
        if constexpr (L::kNW == 0) {
          hipLaunchKernelGGL((norm_fwd_long_kernel<EX, EH, OUT>), dim3(row_grid(R)), dim3(kLongThreads), 0, st, P);
        } else {
          constexpr int per = L::kNW == 1 ? 4 : 1;
          hipLaunchKernelGGL((norm_fwd_kernel<EX, EH, L::kNW, L::kNV, OUT>), dim3(row_grid(ceil_div(R, per))),
                             dim3(L::kNW == 1 ? 256 : 64 * L::kNW), 0, st, P);
        }
      };
      if (out == kInt8)
        go(std::integral_constant<int, kInt8>{});
      else if (out == kE4m3)
        go(std::integral_constant<int, kE4m3>{});
      else
        go(std::integral_constant<int, kSame>{});
      return check_launch("mirl_add_rms_norm_fwd");
    });
  });
}
}  // namespace
}  // namespace mirl

extern "C" int mirl_add_rms_norm_fwd(const void* x, int x_dtype, int64_t ldx, const void* residual, int res_dtype,
                                     int64_t ldr, const void* weight, int w_dtype, int64_t R, int64_t H, double eps,
                                     void* h, void* y, float* y_scale, float* rstd, void* stream) {
  return norm_fwd(y_scale != nullptr ? kE4m3 : kSame, x, x_dtype, ldx, residual, res_dtype, ldr, weight, w_dtype, R, H, eps,
                  h, y, y_scale, rstd, stream);
}

extern "C" int mirl_add_rms_norm_int8_fwd(const void* x, int x_dtype, int64_t ldx, const void* residual, int res_dtype,
                                          int64_t ldr, const void* weight, int w_dtype, int64_t R, int64_t H, double eps,
                                          void* h, int8_t* y, float* y_scale, void* stream) {
  clear_error();
  MIRL_REQUIRE(R <= 0 || y_scale != nullptr, "null pointer argument");
  return norm_fwd(kInt8, x, x_dtype, ldx, residual, res_dtype, ldr, weight, w_dtype, R, H, eps, h, y, y_scale, nullptr, stream);
}

extern "C" int64_t mirl_add_rms_norm_bwd_workspace_elems(int64_t R, int64_t H) {
  if (R <= 0 || H <= 0 || few_rows(R, H)) return 0;
  return (R < kMaxGroups ? R : kMaxGroups) * H;
}

extern "C" int mirl_add_rms_norm_bwd(const void* dy, int x_dtype, int64_t lddy, const void* dh_out, int64_t ldd,
                                     const void* h, int h_dtype, int64_t ldh, const float* rstd, const void* weight,
                                     int w_dtype, int64_t R, int64_t H, void* dx, void* dres, void* dw,
                                     float* workspace, void* stream) {
  clear_error();
  MIRL_REQUIRE(R >= 0 && H > 0 && R < kMaxSide && H < kMaxWidth, "invalid shape R=%lld H=%lld", (long long)R, (long long)H);
  if (int e = check_weight(x_dtype, w_dtype)) return e;
  return with_types(x_dtype, h_dtype, [&](auto ex, auto eh) -> int {
    using EX = decltype(ex);
    using EH = decltype(eh);
    if (R == 0) {
      MIRL_REQUIRE(dw == nullptr, "a weight gradient of no rows");
      return MIRL_OK;
    }
    MIRL_REQUIRE(dy && h && rstd && weight, "null pointer argument");
    MIRL_REQUIRE(R == 1 || (lddy >= H && ldh >= H && (dh_out == nullptr || ldd >= H)),
                 "row strides (%lld, %lld, %lld) are below H=%lld", (long long)lddy, (long long)ldh, (long long)ldd,
                 (long long)H);
    MIRL_REQUIRE(dw == nullptr || workspace != nullptr || mirl_add_rms_norm_bwd_workspace_elems(R, H) == 0,
                 "null pointer argument");
    const int64_t groups = R < kMaxGroups ? R : kMaxGroups;
    const bool few = dw != nullptr && few_rows(R, H);
    NormBwd P{dy, lddy, dh_out, ldd, h, ldh, rstd, Weight{weight, w_dtype == MIRL_DTYPE_F32}, R, H, dx, dres,
              dw != nullptr && !few ? workspace : nullptr, groups, few ? dw : nullptr, 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    with_layout(H, [&](auto layout) -> int {
      using L = decltype(layout);
      if constexpr (L::kNW == 0) {
        if (dx != nullptr || dres != nullptr)
          hipLaunchKernelGGL((norm_bwd_long_kernel<EX, EH>), dim3(row_grid(R)), dim3(kLongThreads), 0, st, P);
        if (dw != nullptr)  // below 2^32 threads: 1024 groups, H < 2^24
          hipLaunchKernelGGL((norm_dw_long_kernel<EX, EH>), dim3((unsigned)(groups * ceil_div(H, 256 * kV))), dim3(256),
                             0, st, P);
      } else {
        constexpr int per = L::kNW == 1 ? 4 : 1;
        P.dw_first = ceil_div(groups, per);
        hipLaunchKernelGGL((norm_bwd_kernel<EX, EH, L::kNW, L::kNV>),
                           dim3((unsigned)(P.dw_first + (few ? ceil_div(H, 16) : 0))),
                           dim3(L::kNW == 1 ? 256 : 64 * L::kNW), 0, st, P);
      }
      return MIRL_OK;
    });
    if (dw != nullptr && !few) {
      auto sum = [&](auto ew) {
        using EW = decltype(ew);
        hipLaunchKernelGGL(norm_dw_sum_kernel<EW>, dim3((unsigned)ceil_div(H, 32)), dim3(1024), 0, st, workspace, groups, H,
                           static_cast<typename EW::raw*>(dw));
      };
      if (w_dtype == MIRL_DTYPE_F32)
        sum(F32{});
      else
        sum(EX{});
    }
    return check_launch("mirl_add_rms_norm_bwd");
  });
}

namespace mirl {
namespace {
template <int OUT>
int quantize(const void* x, int dtype, int64_t ldx, int64_t R, int64_t H, void* y, float* scale, void* stream) {
  clear_error();
  MIRL_REQUIRE(R >= 0 && H > 0 && R < kMaxSide && H < kMaxWidth, "invalid shape R=%lld H=%lld", (long long)R, (long long)H);
  return with_types(dtype, dtype, [&](auto ex, auto) -> int {
    using EX = decltype(ex);
    if (R == 0) return MIRL_OK;
    MIRL_REQUIRE(x && y && scale, "null pointer argument");
    MIRL_REQUIRE(R == 1 || ldx >= H, "row stride %lld is below H=%lld", (long long)ldx, (long long)H);
    hipLaunchKernelGGL((quantize_rows_kernel<EX, OUT>), dim3(row_grid(R)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const typename EX::raw*>(x), ldx, R, H, static_cast<uint8_t*>(y), scale);
    return check_launch("mirl_quantize_rows");
  });
}
}  // namespace
}  // namespace mirl

extern "C" int mirl_quantize_rows(const void* x, int dtype, int64_t ldx, int64_t R, int64_t H, void* y, float* scale,
                                  void* stream) {
  return quantize<kE4m3>(x, dtype, ldx, R, H, y, scale, stream);
}

extern "C" int mirl_quantize_rows_int8(const void* x, int dtype, int64_t ldx, int64_t R, int64_t H, int8_t* y, float* scale,
                                       void* stream) {
  return quantize<kInt8>(x, dtype, ldx, R, H, y, scale, stream);
}
