// What a sampler does to logits before its temperature, top-k and top-p: penalties for repeated
// tokens, biases of single tokens and grammar masks, with the temperature behind them.  Row r of
// sample b follows the first n_b + r of its tokens; for token j with c occurrences behind the prompt,
// `seen` if it occurs at all:
//   z = x + bias;   z = seen ? (z > 0 ? z / rp : z rp) : z;   z = z - freq c - pres [c > 0]
//   y = allowed ? z / T : -inf
// in three forms: y written out (with its backward), y written in place, and the next token's logprob
//   logprob_t = (y_t - M) - log(sum_j exp(y_j - M)),   dx_j = slope_j (onehot_j - p_j) g
// with y never written; slope is what z multiplies x by, over T, 0 where the grammar forbids j.
//
// A workgroup owns a slice of the vocabulary for a run of rows of one sample, and each lane the same
// groups of eight tokens in all of them: it counts the tokens ahead of its first row with LDS atomics
// (whole numbers: their order does not matter), and from then on a row's new token concerns the one
// lane that owns it.  No barrier, sort or table in memory follows the counting, and nothing of size
// [rows, V] is held.  A word per token holds its count, whether it occurred and its bias; a bit per
// token in the lane's registers says whether the word is anything but 0, so that ordinary tokens
// cost one test for a group of eight.

#include "common.h"

#pragma clang fp contract(off)

namespace mirl {
namespace {

constexpr int kG = 8;           // tokens of a lane's group
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

// A token's word: occurrences behind the prompt, whether it occurs in the prompt, 1 + its bias entry.
constexpr uint32_t kCountBits = 20, kInPrompt = 1u << kCountBits, kCount = kInPrompt - 1;
constexpr int kBiasShift = kCountBits + 1;
constexpr int64_t kMaxTokens = kCount, kMaxBias = (int64_t(1) << (32 - kBiasShift)) - 1;

enum Mode { kFwd, kBwd, kApply, kInPlace, kApplyGrad };

struct Params {
  mirl_logit_processors A;
  const void* x;
  int64_t xsb, xsr;
  int64_t B, R, Rt, V;   // rows with a result; rows of the gradient (those past R: zeros)
  int64_t n_vocab;       // ids vs .. vs + n_vocab - 1 stand for the columns
  int64_t slices, chunks;
  int rows;              // rows of a workgroup
  void* y;               // processed logits, or a gradient
  int64_t ysb, ysr;
  const void* dy;        // kApplyGrad
  int64_t gsb, gsr;      // strides of g, or of dy
  const float* g;        // kBwd [B, R]
  const float* stats;    // kBwd [B, R, 2]
  float* part;           // kFwd [B * R, parts, 2]
  float* xt;             // kFwd [B * R]
};

template <class E>
using piece_t = typename Piece<alignof(typename E::raw)>::type;
template <class E>
constexpr int kP = kG / E::kVec;  // 16-byte pieces of a group

template <class E>
__device__ __forceinline__ void unpack_group(const vu4 (&q)[kP<E>], float (&v)[kG]) {
#pragma unroll
  for (int i = 0; i < kP<E>; ++i) {
    float w[E::kVec];
    E::unpack(q[i], w);
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) v[i * E::kVec + e] = w[e];
  }
}
// (rows start anywhere: the hardware takes 16-byte pieces at any element)
template <class E>
__device__ __forceinline__ void load_pieces(const typename E::raw* p, vu4 (&q)[kP<E>]) {
#pragma unroll
  for (int i = 0; i < kP<E>; ++i) q[i] = __builtin_nontemporal_load(reinterpret_cast<const piece_t<E>*>(p) + i);
}
template <class E>
__device__ __forceinline__ void store_group(typename E::raw* row, int64_t c, int64_t V, const float (&v)[kG]) {
  if (c + kG <= V) {
#pragma unroll
    for (int i = 0; i < kP<E>; ++i) {
      float w[E::kVec];
#pragma unroll
      for (int e = 0; e < E::kVec; ++e) w[e] = v[i * E::kVec + e];
      __builtin_nontemporal_store((piece_t<E>)E::pack(w), reinterpret_cast<piece_t<E>*>(row + c) + i);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kG; ++e)
      if (c + e < V) row[c + e] = E::from_float(v[e]);
  }
}
template <class E>
__device__ __forceinline__ void load_tail(const typename E::raw* row, int64_t c, int64_t V, float fill, float (&v)[kG]) {
#pragma unroll
  for (int e = 0; e < kG; ++e) v[e] = c + e < V ? E::load(row + c + e) : fill;
}

// What holds for all rows of a sample.
struct Sample {
  float rp, inv_rp, pres, freq, inv_t;
  const float* bias;
};

// Bias and penalties of the tokens of a group whose bit is set (a wave looks at a token only if one
// of its lanes has it), and with SLOPE what each x was multiplied by.
template <bool SLOPE>
__device__ __forceinline__ void special(float (&v)[kG], float (&slope)[kG], uint32_t bits, const uint32_t* words, const Sample& S) {
#pragma unroll
  for (int e = 0; e < kG; ++e) {
    const bool mine = (bits >> e) & 1u;
    if (__ballot(mine) == 0) continue;
    if (mine) {
      const uint32_t w = words[e];
      float z = v[e];
      if (w >> kBiasShift) z += S.bias[(w >> kBiasShift) - 1];
      if (w & (kInPrompt | kCount)) {
        const float f = z > 0.f ? S.inv_rp : S.rp;
        z *= f;
        if constexpr (SLOPE) slope[e] *= f;
      }
      const uint32_t n = w & kCount;
      z -= S.freq * (float)n;
      z -= n != 0 ? S.pres : 0.f;
      v[e] = z;
    }
  }
}

template <class E, int MODE, int NV>
__global__ __launch_bounds__(kThreads) void processors_kernel(Params P) {
  using raw = typename E::raw;
  constexpr int kSlice = kThreads * NV * kG;
  constexpr bool kReads = MODE != kInPlace;  // every group of a row is read
  __shared__ __align__(16) uint32_t s_word[kSlice];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t slice = blockIdx.x % P.slices, rest = blockIdx.x / P.slices;
  const int64_t chunk = rest % P.chunks, b = rest / P.chunks;
  const int64_t n0 = slice * kSlice, V = P.V;
  const int64_t r0 = chunk * P.rows, r1 = min(r0 + P.rows, P.Rt);
  const mirl_logit_processors& A = P.A;
  const int64_t L = A.n_ids, vs = A.vocab_start;
  const int64_t n_b = A.lengths != nullptr ? A.lengths[b] : 1;
  const int64_t prompt = A.prompt_lengths != nullptr ? A.prompt_lengths[b] : 0;
  const int64_t* ids = A.ids + b * A.ids_stride_b;

  Sample S;
  S.rp = A.repetition != nullptr ? A.repetition[b] : A.repetition_all;
  S.inv_rp = 1.f / S.rp;
  S.pres = A.presence != nullptr ? A.presence[b] : A.presence_all;
  S.freq = A.frequency != nullptr ? A.frequency[b] : A.frequency_all;
  S.inv_t = 1.f / (A.temperature != nullptr ? A.temperature[b] : A.temperature_all);
  S.bias = A.bias + b * A.bias_stride_b;

  // ---- the tokens ahead of row r0 ----
#pragma unroll
  for (int i = 0; i < kSlice / 4 / kThreads; ++i)
    reinterpret_cast<vu4*>(s_word)[i * kThreads + tid] = vu4{0u, 0u, 0u, 0u};
  __syncthreads();
  // the column of an id in this slice, or a number outside it
  auto column = [&](int64_t id) { return id >= vs && id - vs < P.n_vocab ? id - vs - n0 : -1; };
  if (A.n_bias > 0) {  // of two entries of a token the later holds
    for (int64_t k = tid; k < A.n_bias; k += kThreads) {
      const int64_t c = column(A.bias_ids[b * A.bias_stride_b + k]);
      if (c >= 0 && c < kSlice) atomicMax(&s_word[c], (uint32_t)(k + 1) << kBiasShift);
    }
    __syncthreads();
  }
  const int64_t ahead = min(max(n_b + r0, int64_t(0)), L);
  for (int64_t p = tid; p < ahead; p += kThreads) {
    const int64_t c = column(ids[p * A.ids_stride_s]);
    if (c >= 0 && c < kSlice) {
      if (p < prompt)
        atomicOr(&s_word[c], kInPrompt);
      else
        atomicAdd(&s_word[c], 1u);
    }
  }
  __syncthreads();

  // ---- from here on each lane by itself ----
  const int g0 = wave * NV * kWave + lane;  // group u of the lane: g0 + 64 u
  uint32_t bits[(NV + 3) / 4] = {};
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const vu4 a = *reinterpret_cast<const vu4*>(s_word + (g0 + u * kWave) * kG);
    const vu4 c = *reinterpret_cast<const vu4*>(s_word + (g0 + u * kWave) * kG + 4);
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m |= (a[e] != 0 ? 1u << e : 0u) | (c[e] != 0 ? 16u << e : 0u);
    bits[u / 4] |= m << (8 * (u % 4));
  }
  const raw* xb = static_cast<const raw*>(P.x) + b * P.xsb;
  raw* yb = MODE == kFwd ? nullptr : static_cast<raw*>(P.y) + b * P.ysb;
  // rows of the gradient without an upstream one are not read
  auto upstream = [&](int64_t r) { return r < P.R ? P.g[b * P.gsb + r * P.gsr] : 0.f; };
  auto dead_row = [&](int64_t r, float gv) {
    if (gv == 0.f) return true;
    const float* st = P.stats + (b * P.R + r) * 2;
    return st[0] == -INFINITY && st[1] == -INFINITY;  // nothing was left in it
  };
  auto column_of = [&](int u) { return n0 + (int64_t)(g0 + u * kWave) * kG; };
  vu4 q[NV][kP<E>];
  auto issue = [&](int64_t r) {
    const raw* row = MODE == kApplyGrad ? static_cast<const raw*>(P.dy) + b * P.gsb + r * P.gsr : xb + r * P.xsr;
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (column_of(u) + kG <= V) load_pieces<E>(row + column_of(u), q[u]);
  };
  const bool dense = S.inv_t != 1.f;  // kInPlace: every value changes

  float gv = 0.f;
  bool skip = false;
  if constexpr (MODE == kBwd) {
    gv = upstream(r0);
    skip = dead_row(r0, gv);
  }
  if (kReads && !skip) issue(r0);
  for (int64_t r = r0; r < r1; ++r) {
    if (r > r0) {  // the token ahead of this row
      const int64_t p = n_b + r - 1;
      if (p >= 0 && p < L) {
        const int64_t c = column(ids[p * A.ids_stride_s]);
        if (c >= 0 && c < kSlice && (int)(c / (kG * kWave * NV)) == wave) {
          const int in = (int)(c / kG) - wave * NV * kWave;  // 64 u + lane
          if ((in & 63) == lane) {
            s_word[c] = p < prompt ? s_word[c] | kInPrompt : s_word[c] + 1;
#pragma unroll
            for (int u = 0; u < NV; ++u)
              if (u == in / 64) bits[u / 4] |= 1u << (8 * (u % 4) + (int)(c % kG));
          }
        }
      }
    }
    // this row's values, and the next row's on their way
    float v[NV][kG];
    const float g_now = gv;
    const bool skip_now = skip;
    if (kReads && !skip_now) {
      const raw* row = MODE == kApplyGrad ? static_cast<const raw*>(P.dy) + b * P.gsb + r * P.gsr : xb + r * P.xsr;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        if (column_of(u) + kG <= V)
          unpack_group<E>(q[u], v[u]);
        else
          load_tail<E>(row, column_of(u), V, MODE == kFwd ? -INFINITY : 0.f, v[u]);
      }
    }
    if (r + 1 < r1) {
      if constexpr (MODE == kBwd) {
        gv = upstream(r + 1);
        skip = dead_row(r + 1, gv);
      }
      if (kReads && !skip) issue(r + 1);
    }
    raw* yr = MODE == kFwd ? nullptr : yb + r * P.ysr;
    if constexpr (MODE == kBwd) {
      if (skip_now) {
        const float z[kG] = {};
#pragma unroll
        for (int u = 0; u < NV; ++u)
          if (column_of(u) < V) store_group<E>(yr, column_of(u), V, z);
        continue;
      }
    }
    const uint8_t* mask = nullptr;
    if (A.n_masks > 0) {
      const int64_t m = A.mask_rows[b * A.mask_rows_stride_b + r * A.mask_rows_stride_r];
      if (m >= 0 && m < A.n_masks) mask = reinterpret_cast<const uint8_t*>(A.masks + m * A.mask_stride);
    }
    uint32_t allowed[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      allowed[u] = 0xffu;
      if (mask != nullptr && column_of(u) < V) allowed[u] = mask[column_of(u) / kG];
    }
    // the next token's place in this wave: group of the lane, and which of its eight
    int tu = -1, tlane = -1, te = -1;
    if constexpr (MODE == kFwd || MODE == kBwd) {
      const int64_t p = n_b + r;
      const int64_t c = p >= 0 && p < L ? column(ids[p * A.ids_stride_s]) : -1;
      if (c >= 0 && c < kSlice && (int)(c / (kG * kWave * NV)) == wave) {
        const int in = (int)(c / kG) - wave * NV * kWave;
        tu = in / 64;
        tlane = in & 63;
        te = (int)(c % kG);
      }
    }
    float none[kG];
    if constexpr (MODE == kFwd) {
      float m = -INFINITY;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const uint32_t sp = (bits[u / 4] >> (8 * (u % 4))) & 0xffu;
        if (__ballot(sp != 0)) special<false>(v[u], none, sp, s_word + (g0 + u * kWave) * kG, S);
        if (__ballot(allowed[u] != 0xffu)) {
#pragma unroll
          for (int e = 0; e < kG; ++e) v[u][e] = (allowed[u] >> e) & 1u ? v[u][e] : -INFINITY;
        }
        if (u == tu && lane == tlane) {
          float t = 0.f;
#pragma unroll
          for (int e = 0; e < kG; ++e) t = e == te ? v[u][e] : t;
          P.xt[b * P.R + r] = t;
        }
#pragma unroll
        for (int e = 0; e < kG; ++e) m = fmaxf(m, v[u][e]);
      }
      // the lane's sum, then the wave's: sums of 2^(y c - fl(m c)) with c = log2(e) / T
      const float c = kLog2e * S.inv_t;
      const float M = wave_max(m);
      const float off = M * c;
      float s4[4] = {0.f, 0.f, 0.f, 0.f};
      const bool in_range = fabsf(off) < INFINITY;
      if (in_range) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
          for (int e = 0; e < kG; ++e) s4[e & 3] += fast_exp2(fmaf(v[u][e], c, -off));
      } else if (M != -INFINITY) {  // a row of nothing but the type's lowest values, or of an infinity
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
          for (int e = 0; e < kG; ++e) s4[e & 3] += fast_exp2((v[u][e] - M) * c);
      } else {  // -inf, and NaN, which a maximum does not show
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
          for (int e = 0; e < kG; ++e) s4[e & 3] = v[u][e] != v[u][e] ? v[u][e] : s4[e & 3];
      }
      float s = wave_sum((s4[0] + s4[1]) + (s4[2] + s4[3]));
      if (in_range) s *= fast_exp2(-fmaf(M, c, -off));  // the offset's rounding undone
      if (lane == 0) {
        float* dst = P.part + ((b * P.R + r) * (P.slices * kWaves) + slice * kWaves + wave) * 2;
        dst[0] = M;
        dst[1] = s;
      }
    } else if constexpr (MODE == kBwd) {
      const float* st = P.stats + (b * P.R + r) * 2;
      const float M = st[0], c = kLog2e * S.inv_t, ls = st[1] * kLog2e, gt = g_now * S.inv_t;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        if (column_of(u) >= V) continue;
        const uint32_t sp = (bits[u / 4] >> (8 * (u % 4))) & 0xffu;
        float slope[kG];
        const bool any = __ballot(sp != 0) != 0;
        if (any) {
#pragma unroll
          for (int e = 0; e < kG; ++e) slope[e] = 1.f;
          special<true>(v[u], slope, sp, s_word + (g0 + u * kWave) * kG, S);
        }
        const bool masked = __ballot(allowed[u] != 0xffu) != 0;
        float o[kG];
#pragma unroll
        for (int e = 0; e < kG; ++e) o[e] = -fast_exp2(fmaf(v[u][e] - M, c, -ls)) * gt;
        if (u == tu && lane == tlane) {
#pragma unroll
          for (int e = 0; e < kG; ++e) o[e] = e == te ? (1.f - fast_exp2(fmaf(v[u][e] - M, c, -ls))) * gt : o[e];
        }
        if (any) {
#pragma unroll
          for (int e = 0; e < kG; ++e) o[e] *= slope[e];
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < kG; ++e) o[e] = (allowed[u] >> e) & 1u ? o[e] : 0.f;
        }
        store_group<E>(yr, column_of(u), V, o);
      }
    } else {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int64_t c = column_of(u);
        if (c >= V) continue;
        const uint32_t sp = (bits[u / 4] >> (8 * (u % 4))) & 0xffu;
        if constexpr (MODE == kInPlace) {
          if (!dense && sp == 0 && allowed[u] == 0xffu) continue;
          if (c + kG <= V) {
            vu4 w[kP<E>];
            load_pieces<E>(xb + r * P.xsr + c, w);
            unpack_group<E>(w, v[u]);
          } else {
            load_tail<E>(xb + r * P.xsr, c, V, 0.f, v[u]);
          }
        }
        float slope[kG];
        if constexpr (MODE == kApplyGrad) {
#pragma unroll
          for (int e = 0; e < kG; ++e) slope[e] = S.inv_t;
          if (sp != 0) {
            float xv[kG];
            if (c + kG <= V) {
              vu4 w[kP<E>];
              load_pieces<E>(xb + r * P.xsr + c, w);
              unpack_group<E>(w, xv);
            } else {
              load_tail<E>(xb + r * P.xsr, c, V, 0.f, xv);
            }
            special<true>(xv, slope, sp, s_word + (g0 + u * kWave) * kG, S);
          }
#pragma unroll
          for (int e = 0; e < kG; ++e) v[u][e] = (allowed[u] >> e) & 1u ? v[u][e] * slope[e] : 0.f;
        } else {
          if (__ballot(sp != 0)) special<false>(v[u], slope, sp, s_word + (g0 + u * kWave) * kG, S);
#pragma unroll
          for (int e = 0; e < kG; ++e) v[u][e] = (allowed[u] >> e) & 1u ? v[u][e] * S.inv_t : -INFINITY;
        }
        store_group<E>(yr, c, V, v[u]);
      }
    }
  }
}

// Per row, one wave: the slices' partials joined, the next token's logprob.
__global__ __launch_bounds__(kThreads) void processors_join_kernel(Params P, float* out, float* stats) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= P.B * P.R) return;
  const int64_t b = row / P.R, r = row - b * P.R, n = P.slices * kWaves;
  const mirl_logit_processors& A = P.A;
  const float inv_t = 1.f / (A.temperature != nullptr ? A.temperature[b] : A.temperature_all), c = kLog2e * inv_t;
  const float* p = P.part + row * n * 2;
  float M = -INFINITY, s = 0.f;
  for (int64_t j = lane; j < n; j += kWave) M = fmaxf(M, p[2 * j]);
  M = wave_max(M);
  for (int64_t j = lane; j < n; j += kWave) {
    const float mj = p[2 * j], sj = p[2 * j + 1];
    // (a part with nothing in it has a sum of 0; one of NaN has a maximum of -inf too, and NaN as its sum)
    if (mj != -INFINITY)
      s += sj * fast_exp2((mj - M) * c);
    else if (sj != 0.f)
      s = sj;
  }
  s = wave_sum(s);
  if (lane != 0) return;
  const int64_t n_b = A.lengths != nullptr ? A.lengths[b] : 1, at = n_b + r;
  const int64_t t = at >= 0 && at < A.n_ids ? A.ids[b * A.ids_stride_b + at * A.ids_stride_s] - A.vocab_start : -1;
  const float logsum = logf(s);
  float lp = 0.f;
  if (t >= 0 && t < P.n_vocab) lp = M == -INFINITY && s == 0.f ? -INFINITY : (P.xt[row] - M) * inv_t - logsum;
  out[row] = lp;
  if (stats != nullptr) {
    stats[2 * row] = M;
    stats[2 * row + 1] = logsum;
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Groups of a lane and rows of a workgroup.
struct Plan {
  int nv;
  int64_t slices, rows, chunks;
};
Plan plan_of(int64_t B, int64_t R, int64_t V) {
  Plan p;
  p.nv = B * R * ceil_div(V, kThreads * kG) >= 4 * 4096 ? 4 : 1;
  p.slices = ceil_div(V, kThreads * kG * p.nv);
  p.rows = 32;
  while (p.rows > 1 && B * ceil_div(R, p.rows) * p.slices < 2048) p.rows /= 2;
  while (B * ceil_div(R, p.rows) * p.slices >= (int64_t(1) << 24)) p.rows *= 2;
  p.chunks = ceil_div(R, p.rows);
  return p;
}

template <int MODE>
int launch(Params& P, int dtype, int64_t rows, const char* what, hipStream_t st) {
  const Plan p = plan_of(P.B, rows, P.V);
  P.slices = p.slices;
  P.chunks = p.chunks;
  P.rows = (int)p.rows;
  const dim3 grid((unsigned)(P.B * p.chunks * p.slices)), block(kThreads);
  auto go = [&](auto e) {
    using E = decltype(e);
    if (p.nv == 4)
      hipLaunchKernelGGL((processors_kernel<E, MODE, 4>), grid, block, 0, st, P);
    else
      hipLaunchKernelGGL((processors_kernel<E, MODE, 1>), grid, block, 0, st, P);
  };
  if (dtype == MIRL_DTYPE_F32)
    go(F32{});
  else if (dtype == MIRL_DTYPE_BF16)
    go(BF16{});
  else
    go(F16{});
  return check_launch(what);
}

int check_args(const mirl_logit_processors* A, int dtype, int64_t B, int64_t R, int64_t V) {
  MIRL_REQUIRE(dtype == MIRL_DTYPE_F32 || dtype == MIRL_DTYPE_BF16 || dtype == MIRL_DTYPE_F16,
               "unsupported logits dtype code %d", dtype);
  MIRL_REQUIRE(A != nullptr, "null pointer argument");
  MIRL_REQUIRE(B >= 0 && R >= 0 && V > 0, "invalid shape B=%lld R=%lld V=%lld", (long long)B, (long long)R, (long long)V);
  MIRL_REQUIRE(V < (int64_t(1) << 31) && B * R < (int64_t(1) << 31), "sizes exceed 2^31-1");
  MIRL_REQUIRE(A->n_ids >= 0 && A->n_ids <= kMaxTokens, "%lld tokens of a sample, at most %lld are counted",
               (long long)A->n_ids, (long long)kMaxTokens);
  MIRL_REQUIRE(A->n_bias >= 0 && A->n_bias <= kMaxBias, "%lld biases of a sample, at most %lld are held",
               (long long)A->n_bias, (long long)kMaxBias);
  MIRL_REQUIRE(A->n_masks >= 0 && (A->n_masks == 0 || A->mask_stride >= ceil_div(V, 32)),
               "grammar masks of %lld words do not cover %lld columns", (long long)A->mask_stride, (long long)V);
  if (B * R == 0) return MIRL_OK;
  MIRL_REQUIRE((A->n_ids == 0 || A->ids != nullptr) && (A->n_bias == 0 || (A->bias_ids != nullptr && A->bias != nullptr)) &&
                   (A->n_masks == 0 || (A->masks != nullptr && A->mask_rows != nullptr)),
               "null pointer argument");
  return MIRL_OK;
}

Params params_of(const mirl_logit_processors* A, const void* x, int64_t B, int64_t R, int64_t Rt, int64_t V, int64_t xsb,
                 int64_t xsr) {
  Params P{};
  P.A = *A;
  P.x = x;
  P.B = B;
  P.R = R;
  P.Rt = Rt;
  P.V = V;
  P.xsb = xsb;
  P.xsr = xsr;
  const int64_t n = A->vocab_end - A->vocab_start;
  P.n_vocab = n < V ? n : V;
  return P;
}

}  // namespace
}  // namespace mirl

using namespace mirl;

extern "C" int64_t mirl_processed_logprob_workspace_elems(int64_t B, int64_t R, int64_t V) {
  if (B <= 0 || R <= 0 || V <= 0) return 0;
  return B * R * (plan_of(B, R, V).slices * kWaves * 2 + 1);
}

extern "C" int mirl_processed_logprob_fwd(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                          int64_t stride_r, const mirl_logit_processors* processors, float* out,
                                          float* stats, float* workspace, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, R, V)) return e;
  if (B * R == 0) return MIRL_OK;
  MIRL_REQUIRE(logits && out && workspace, "null pointer argument");
  Params P = params_of(processors, logits, B, R, R, V, stride_b, stride_r);
  hipStream_t st = static_cast<hipStream_t>(stream);
  P.part = workspace;
  P.xt = workspace + B * R * plan_of(B, R, V).slices * kWaves * 2;
  if (int e = launch<kFwd>(P, dtype, R, "mirl_processed_logprob_fwd", st)) return e;
  hipLaunchKernelGGL(processors_join_kernel, dim3((unsigned)ceil_div(B * R, kWaves)), dim3(kThreads), 0, st, P, out, stats);
  return check_launch("mirl_processed_logprob_fwd");
}

extern "C" int mirl_processed_logprob_bwd(const void* logits, int dtype, int64_t B, int64_t R, int64_t Rt, int64_t V,
                                          int64_t stride_b, int64_t stride_r, const mirl_logit_processors* processors,
                                          const float* stats, const float* grad_out, int64_t g_stride_b, int64_t g_stride_r,
                                          void* grad_in, int64_t gi_stride_b, int64_t gi_stride_r, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, Rt, V)) return e;
  MIRL_REQUIRE(R >= 0 && R <= Rt, "invalid shape R=%lld of %lld rows", (long long)R, (long long)Rt);
  if (B * Rt == 0) return MIRL_OK;
  MIRL_REQUIRE(logits && grad_in && (R == 0 || (stats && grad_out)), "null pointer argument");
  Params P = params_of(processors, logits, B, R, Rt, V, stride_b, stride_r);
  P.stats = stats;
  P.g = grad_out;
  P.gsb = g_stride_b;
  P.gsr = g_stride_r;
  P.y = grad_in;
  P.ysb = gi_stride_b;
  P.ysr = gi_stride_r;
  return launch<kBwd>(P, dtype, Rt, "mirl_processed_logprob_bwd", static_cast<hipStream_t>(stream));
}

extern "C" int mirl_process_logits(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                   int64_t stride_r, const mirl_logit_processors* processors, void* out,
                                   int64_t o_stride_b, int64_t o_stride_r, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, R, V)) return e;
  if (B * R == 0) return MIRL_OK;
  MIRL_REQUIRE(logits && out, "null pointer argument");
  MIRL_REQUIRE(out != logits || (o_stride_b == stride_b && o_stride_r == stride_r), "in place, the strides are those of the logits");
  Params P = params_of(processors, logits, B, R, R, V, stride_b, stride_r);
  P.y = out;
  P.ysb = o_stride_b;
  P.ysr = o_stride_r;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return out == logits ? launch<kInPlace>(P, dtype, R, "mirl_process_logits", st)
                       : launch<kApply>(P, dtype, R, "mirl_process_logits", st);
}

extern "C" int mirl_process_logits_bwd(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                       int64_t stride_r, const mirl_logit_processors* processors, const void* grad_out,
                                       int64_t g_stride_b, int64_t g_stride_r, void* grad_in, int64_t gi_stride_b,
                                       int64_t gi_stride_r, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, R, V)) return e;
  if (B * R == 0) return MIRL_OK;
  MIRL_REQUIRE(logits && grad_out && grad_in, "null pointer argument");
  Params P = params_of(processors, logits, B, R, R, V, stride_b, stride_r);
  P.dy = grad_out;
  P.gsb = g_stride_b;
  P.gsr = g_stride_r;
  P.y = grad_in;
  P.ysb = gi_stride_b;
  P.ysr = gi_stride_r;
  return launch<kApplyGrad>(P, dtype, R, "mirl_process_logits_bwd", static_cast<hipStream_t>(stream));
}
