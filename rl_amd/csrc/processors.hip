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
constexpr uint32_t kGroupBytes = kG * sizeof(typename E::raw);

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
// A group at `at` bytes into a row's slice (rows start anywhere: the hardware takes 16-byte pieces at
// any element).
template <class E>
__device__ __forceinline__ void load_group(const typename E::raw* slice, uint32_t at, vu4 (&q)[kP<E>]) {
#pragma unroll
  for (int i = 0; i < kP<E>; ++i)
    q[i] = __builtin_nontemporal_load(reinterpret_cast<const piece_t<E>*>(reinterpret_cast<const char*>(slice) + at) + i);
}
template <class E>
__device__ __forceinline__ void store_group(typename E::raw* slice, uint32_t at, const float (&v)[kG]) {
#pragma unroll
  for (int i = 0; i < kP<E>; ++i) {
    float w[E::kVec];
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) w[e] = v[i * E::kVec + e];
    __builtin_nontemporal_store((piece_t<E>)E::pack(w), reinterpret_cast<piece_t<E>*>(reinterpret_cast<char*>(slice) + at) + i);
  }
}

// The maximum and the sum over a wave by lane permutes within the VALU (64 lanes; in lane 63, given to all).
template <int CTRL>
__device__ __forceinline__ float from_lane(float other, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(other), __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <class F>
__device__ __forceinline__ float wave_fold(float v, float none, F&& f) {
  v = f(v, from_lane<0x111>(none, v));  // row_shr 1, 2, 4, 8
  v = f(v, from_lane<0x112>(none, v));
  v = f(v, from_lane<0x114>(none, v));
  v = f(v, from_lane<0x118>(none, v));
  v = f(v, from_lane<0x142>(none, v));  // row_bcast 15, 31
  v = f(v, from_lane<0x143>(none, v));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float of_row(float v, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i)); }

// What holds for all rows of a sample.
struct Sample {
  float rp, inv_rp, pres, freq, inv_t;
  const float* bias;
};

// Bias and penalties of a group's tokens: those of any lane of the wave (`any`, a scalar), in the
// lanes that have them (`bits`); with SLOPE what each x was multiplied by.
template <bool SLOPE>
__device__ __forceinline__ void special(float (&v)[kG], float (&slope)[kG], uint32_t any, uint32_t bits, const vu4* words,
                                        const Sample& S) {
#pragma unroll
  for (int e = 0; e < kG; ++e) {
    if ((any & (1u << e)) == 0) continue;
    if ((bits >> e) & 1u) {
      const uint32_t w = words[e / 4][e % 4];
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
  constexpr int kWaveCols = kWave * NV * kG, kSlice = kWaves * kWaveCols;
  __shared__ __align__(16) uint32_t s_word[kSlice];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t slices = (uint32_t)P.slices, chunks = (uint32_t)P.chunks;
  const uint32_t slice = blockIdx.x % slices, rest = blockIdx.x / slices;
  const uint32_t chunk = rest % chunks, b = rest / chunks;
  const int64_t n0 = (int64_t)slice * kSlice;
  const int64_t r0 = (int64_t)chunk * P.rows;
  const int n_rows = (int)min((int64_t)P.rows, P.Rt - r0);
  const mirl_logit_processors& A = P.A;
  const int64_t L = A.n_ids;
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
  // an id's column in this slice, or -1
  const int64_t first_id = A.vocab_start + n0;
  const uint32_t here = (uint32_t)max(int64_t(0), min((int64_t)kSlice, P.n_vocab - n0));
  auto column = [&](int64_t id) {
    const uint64_t c = (uint64_t)id - (uint64_t)first_id;
    return c < here ? (int)c : -1;
  };
  __syncthreads();
  if (A.n_bias > 0) {  // of two entries of a token the later holds
    for (int64_t k = tid; k < A.n_bias; k += kThreads) {
      const int c = column(A.bias_ids[b * A.bias_stride_b + k]);
      if (c >= 0) atomicMax(&s_word[c], (uint32_t)(k + 1) << kBiasShift);
    }
    __syncthreads();
  }
  const int ahead = (int)min(max(n_b + r0, int64_t(0)), L);
  const int in_prompt = (int)min(max(prompt, int64_t(0)), L);
#pragma unroll 4
  for (int p = tid; p < ahead; p += kThreads) {
    const int c = column(ids[p * A.ids_stride_s]);
    if (c >= 0) {
      if (p < in_prompt)
        atomicOr(&s_word[c], kInPrompt);
      else
        atomicAdd(&s_word[c], 1u);
    }
  }
  // What the rows need, row r0 + l in lane l: the token that is new ahead of it and the one behind it
  // (columns of this wave, or -1), its mask, its gradient and statistics.
  int m_new = -1, m_next = -1, m_mask = -1;
  float m_g = 0.f, m_M = 0.f, m_ls = 0.f;
  if (lane < n_rows) {
    const int64_t r = r0 + lane, at = n_b + r;
    auto of_wave = [&](int c) { return c >= 0 && c / kWaveCols == wave ? c - wave * kWaveCols : -1; };
    if (lane > 0 && at > 0 && at <= L) {
      m_new = of_wave(column(ids[(at - 1) * A.ids_stride_s]));
      if (m_new >= 0 && at - 1 < prompt) m_new |= 1 << 30;
    }
    if constexpr (MODE == kFwd || MODE == kBwd) {
      if (at >= 0 && at < L) m_next = of_wave(column(ids[at * A.ids_stride_s]));
    }
    if (A.n_masks > 0 && (MODE != kBwd || r < P.R)) {
      const int64_t m = A.mask_rows[b * A.mask_rows_stride_b + r * A.mask_rows_stride_r];
      m_mask = m >= 0 && m < A.n_masks ? (int)m : -1;
    }
    if constexpr (MODE == kBwd) {
      if (r < P.R) {
        m_g = P.g[b * P.gsb + r * P.gsr];
        m_M = P.stats[(b * P.R + r) * 2];
        m_ls = P.stats[(b * P.R + r) * 2 + 1];
        if (m_M == -INFINITY && m_ls == -INFINITY) m_g = 0.f;  // nothing was left in the row
      }
    }
  }
  __syncthreads();

  // ---- from here on each wave by itself ----
  const int g0 = wave * NV * kWave + lane;  // group u of the lane: g0 + 64 u
  const vu4* words = reinterpret_cast<const vu4*>(s_word) + g0 * (kG / 4);
  constexpr int kU = kWave * (kG / 4);  // between the lane's groups
  uint32_t bits[(NV + 3) / 4] = {}, any[(NV + 3) / 4] = {};  // a byte per group: the lane's, the wave's
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const vu4 lo = words[u * kU], hi = words[u * kU + 1];
#pragma unroll
    for (int e = 0; e < kG; ++e) {
      const bool set = (e < 4 ? lo[e & 3] : hi[e & 3]) != 0;
      bits[u / 4] |= set ? 1u << (8 * (u % 4) + e) : 0u;
      any[u / 4] |= __ballot(set) != 0 ? 1u << (8 * (u % 4) + e) : 0u;
    }
  }
  const raw* xr = static_cast<const raw*>(P.x) + b * P.xsb + r0 * P.xsr + n0;
  const raw* dyr = MODE == kApplyGrad ? static_cast<const raw*>(P.dy) + b * P.gsb + r0 * P.gsr + n0 : nullptr;
  raw* yr = MODE == kFwd ? nullptr : static_cast<raw*>(P.y) + b * P.ysb + r0 * P.ysr + n0;
  const uint32_t left = (uint32_t)min((int64_t)kSlice, P.V - n0);  // columns of the slice
  const uint32_t at0 = g0 * kGroupBytes<E>;
  const bool dense = S.inv_t != 1.f;  // kInPlace: every value changes

  // WHOLE: the slice lies inside the row
  auto rows = [&](auto whole_c) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole_c)::value;
    constexpr bool kStreams = MODE != kInPlace;  // every group of a row is read
    auto full = [&](int u) { return WHOLE || (uint32_t)(g0 + u * kWave + 1) * kG <= left; };
    auto at = [&](int u) { return at0 + u * kWave * kGroupBytes<E>; };
    auto tail = [&](const raw* row, int u, float fill, float (&v)[kG]) {
#pragma unroll
      for (int e = 0; e < kG; ++e) {
        const uint32_t c = (uint32_t)(g0 + u * kWave) * kG + e;
        v[e] = c < left ? E::load(row + c) : fill;
      }
    };
    auto put = [&](int u, const float (&v)[kG]) {
      if (full(u)) {
        store_group<E>(yr, at(u), v);
      } else {
#pragma unroll
        for (int e = 0; e < kG; ++e) {
          const uint32_t c = (uint32_t)(g0 + u * kWave) * kG + e;
          if (c < left) yr[c] = E::from_float(v[e]);
        }
      }
    };
    vu4 q[NV][kP<E>];
    auto issue = [&](const raw* row, int u) {
      if (full(u)) load_group<E>(row, at(u), q[u]);
    };
    bool read = true;  // whether this row's values are on their way
    if constexpr (MODE == kBwd) read = of_row(m_g, 0) != 0.f;
    if (kStreams && read) {
#pragma unroll
      for (int u = 0; u < NV; ++u) issue(MODE == kApplyGrad ? dyr : xr, u);
    }
    for (int i = 0; i < n_rows; ++i) {
      if (i > 0) {  // the token ahead of this row
        const int t = __builtin_amdgcn_readlane(m_new, i);
        if (t >= 0) {
          const uint32_t c = (uint32_t)t & ((1u << 30) - 1), group = c / kG, e = c % kG;
          const uint32_t bit = 1u << e;
          if ((int)(group % kWave) == lane) {
            uint32_t& w = s_word[wave * kWaveCols + c];
            w = (uint32_t)t >> 30 ? w | kInPrompt : w + 1;
          }
#pragma unroll
          for (int u = 0; u < NV; ++u)
            if ((int)(group / kWave) == u) {
              any[u / 4] |= bit << (8 * (u % 4));
              if ((int)(group % kWave) == lane) bits[u / 4] |= bit << (8 * (u % 4));
            }
        }
      }
      const bool more = i + 1 < n_rows;
      const raw* next = MODE == kApplyGrad ? dyr + P.gsr : xr + P.xsr;
      float g_now = 0.f, M_now = 0.f, ls_now = 0.f;
      bool read_next = more;
      if constexpr (MODE == kBwd) {
        g_now = of_row(m_g, i);
        M_now = of_row(m_M, i);
        ls_now = of_row(m_ls, i);
        read_next = more && of_row(m_g, more ? i + 1 : i) != 0.f;
      }
      // the next token's group of the lane, and which of its eight
      int tu = -1, tlane = -1, te = -1;
      if constexpr (MODE == kFwd || MODE == kBwd) {
        const int t = __builtin_amdgcn_readlane(m_next, i);
        if (t >= 0) {
          tu = t / (kG * kWave);
          tlane = t / kG % kWave;
          te = t % kG;
        }
      }
      const int m = __builtin_amdgcn_readlane(m_mask, i);
      uint32_t allowed[NV];
#pragma unroll
      for (int u = 0; u < NV; ++u) allowed[u] = 0xffu;
      if (m >= 0) {
        const uint8_t* mask = reinterpret_cast<const uint8_t*>(A.masks + (int64_t)m * A.mask_stride) + n0 / kG;
#pragma unroll
        for (int u = 0; u < NV; ++u)
          if (WHOLE || (uint32_t)(g0 + u * kWave) * kG < left) allowed[u] = mask[(uint32_t)(g0 + u * kWave)];
      }
      auto wave_bits = [&](int u) { return (any[u / 4] >> (8 * (u % 4))) & 0xffu; };
      auto lane_bits = [&](int u) { return (bits[u / 4] >> (8 * (u % 4))) & 0xffu; };
      // group u of this row, and the next row's on its way
      auto take = [&](int u, float fill, float (&v)[kG]) {
        if (full(u))
          unpack_group<E>(q[u], v);
        else
          tail(MODE == kApplyGrad ? dyr : xr, u, fill, v);
        if (read_next) issue(next, u);
      };
      if constexpr (MODE == kFwd) {
        float v[NV][kG], none[kG];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          take(u, -INFINITY, v[u]);
          if (wave_bits(u) != 0) special<false>(v[u], none, wave_bits(u), lane_bits(u), words + u * kU, S);
          if (m >= 0) {
#pragma unroll
            for (int e = 0; e < kG; ++e) v[u][e] = (allowed[u] >> e) & 1u ? v[u][e] : -INFINITY;
          }
          if (u == tu) {
            float t = v[u][0];
#pragma unroll
            for (int e = 1; e < kG; ++e) t = e == te ? v[u][e] : t;
            if (lane == tlane) P.xt[b * P.R + r0 + i] = t;
          }
#pragma unroll
          for (int e = 0; e < kG; ++e) mx = fmaxf(mx, v[u][e]);
        }
        // sums of 2^(y c - fl(M c)) with c = log2(e) / T, M the wave's maximum
        const float c = kLog2e * S.inv_t;
        const float M = wave_fold(mx, -INFINITY, [](float x, float y) { return fmaxf(x, y); });
        const float off = M * c;
        const bool in_range = fabsf(off) < INFINITY;
        float s4[4] = {0.f, 0.f, 0.f, 0.f};
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
        float s = wave_fold((s4[0] + s4[1]) + (s4[2] + s4[3]), 0.f, [](float x, float y) { return x + y; });
        if (in_range) s *= fast_exp2(-fmaf(M, c, -off));  // the offset's rounding undone
        if (lane == 0)
          reinterpret_cast<float2*>(P.part)[(b * P.R + r0 + i) * (P.slices * kWaves) + slice * kWaves + wave] = float2{M, s};
      } else if constexpr (MODE == kBwd) {
        if (g_now == 0.f) {
          const float z[kG] = {};
#pragma unroll
          for (int u = 0; u < NV; ++u) {
            put(u, z);
            if (read_next) issue(next, u);
          }
        } else {
          const float c = kLog2e * S.inv_t, ls = ls_now * kLog2e, gt = g_now * S.inv_t;
#pragma unroll
          for (int u = 0; u < NV; ++u) {
            float v[kG], o[kG], slope[kG];
            take(u, 0.f, v);
#pragma unroll
            for (int e = 0; e < kG; ++e) slope[e] = 1.f;
            if (wave_bits(u) != 0) special<true>(v, slope, wave_bits(u), lane_bits(u), words + u * kU, S);
#pragma unroll
            for (int e = 0; e < kG; ++e) o[e] = fast_exp2(fmaf(v[e] - M_now, c, -ls)) * -gt;
            if (u == tu) {
#pragma unroll
              for (int e = 0; e < kG; ++e)
                o[e] = lane == tlane && e == te ? (1.f - fast_exp2(fmaf(v[e] - M_now, c, -ls))) * gt : o[e];
            }
            if (wave_bits(u) != 0) {
#pragma unroll
              for (int e = 0; e < kG; ++e) o[e] *= slope[e];
            }
            if (m >= 0) {
#pragma unroll
              for (int e = 0; e < kG; ++e) o[e] = (allowed[u] >> e) & 1u ? o[e] : 0.f;
            }
            put(u, o);
          }
        }
      } else if constexpr (MODE == kApply) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          float v[kG], none[kG];
          take(u, 0.f, v);
          if (wave_bits(u) != 0) special<false>(v, none, wave_bits(u), lane_bits(u), words + u * kU, S);
#pragma unroll
          for (int e = 0; e < kG; ++e) v[e] *= S.inv_t;
          if (m >= 0) {
#pragma unroll
            for (int e = 0; e < kG; ++e) v[e] = (allowed[u] >> e) & 1u ? v[e] : -INFINITY;
          }
          put(u, v);
        }
      } else {
        // these read the logits of some groups only
        auto logits_of = [&](int u, float (&v)[kG]) {
          if (full(u)) {
            vu4 w[kP<E>];
            load_group<E>(xr, at(u), w);
            unpack_group<E>(w, v);
          } else {
            tail(xr, u, 0.f, v);
          }
        };
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          float v[kG], slope[kG];
          if constexpr (MODE == kInPlace) {
            const bool mine = dense || lane_bits(u) != 0 || allowed[u] != 0xffu;
            if (mine) {
              logits_of(u, v);
              special<false>(v, slope, 0xffu, lane_bits(u), words + u * kU, S);
#pragma unroll
              for (int e = 0; e < kG; ++e) v[e] = (allowed[u] >> e) & 1u ? v[e] * S.inv_t : -INFINITY;
              put(u, v);
            }
          } else {
            take(u, 0.f, v);
#pragma unroll
            for (int e = 0; e < kG; ++e) slope[e] = S.inv_t;
            if (wave_bits(u) != 0 && lane_bits(u) != 0) {
              float x[kG];
              logits_of(u, x);
              special<true>(x, slope, wave_bits(u), lane_bits(u), words + u * kU, S);
            }
#pragma unroll
            for (int e = 0; e < kG; ++e) v[e] *= slope[e];
            if (m >= 0) {
#pragma unroll
              for (int e = 0; e < kG; ++e) v[e] = (allowed[u] >> e) & 1u ? v[e] : 0.f;
            }
            put(u, v);
          }
        }
      }
      read = read_next;
      xr += P.xsr;
      if (MODE == kApplyGrad) dyr += P.gsr;
      if (MODE != kFwd) yr += P.ysr;
    }
  };
  if (left == kSlice)
    rows(std::true_type{});
  else
    rows(std::false_type{});
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
