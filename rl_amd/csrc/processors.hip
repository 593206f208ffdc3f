// What a sampler does to logits before its temperature, top-k and top-p: penalties for repeated
// tokens, biases of single tokens and grammar masks, with the temperature behind them.  Row r of
// sample b follows the first n_b + r of its tokens; for token j with c occurrences behind the prompt,
// `seen` if it occurs at all:
//   z = x + bias;   z = seen ? (z > 0 ? z / rp : z rp) : z;   z = z - freq c - pres [c > 0]
//   y = allowed ? z / T : -inf
// in three forms: y written out in the logits' type, or in fp32 for a filter (either with its backward), y written in
// place, and the next token's logprob
//   logprob_t = (y_t - M) - log(sum_j exp(y_j - M)),   dx_j = slope_j (onehot_j - p_j) g
// with y never written; slope is what z multiplies x by, over T, 0 where the grammar forbids j.
//
// A first launch puts each sample's tokens, 4096 at a time, and its biases into buckets by 2048 columns
// (processors_table_kernel).
// A workgroup then owns a slice of the vocabulary, one or more buckets, for a run of rows of one sample,
// and each lane the same groups of eight tokens in all of them: it counts the bucket's tokens ahead of its
// first row with LDS atomics (whole numbers: their order does not matter), and from then on a row's
// new token concerns the one lane that owns it.  No barrier follows the counting, and nothing of size
// [rows, V] is held.  A word per token holds its count, whether it occurred and its bias; a bit per
// token in the lane's registers says whether the word is anything but 0, so that ordinary tokens
// cost one test for a group of eight.
//
// Bound by memory but for the logprobs' forward, which the vector units share (some 60 instructions for eight
// ordinary values of bf16).  bf16 [8, 2048, 151936] with the penalties and biases of a GRPO step, half of the rows without
// a gradient: forward 920 us (4.98 GB, 5.4 TB/s; 860 where no token of the rows occurs, logprob.hip's of untouched
// logits 730), backward 1.36 to 1.43 ms (7.4 GB, 5.3 TB/s; logprob.hip's 1.22).  [2, 2048, 151936]: written out
// 412 us (2.49 GB, 6.0 TB/s), its backward 495 (5.0; the logits of tokens that occur are read as well); in fp32 810 us
// (3.73 GB, 4.6 TB/s), its backward 733 (5.1).  One token of each of 64 requests behind up to 2048 tokens: table 7 us,
// logprobs 14 and 4 to join, written out 16, in place 14: the latency of a few loads that wait for each other.

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

// The table of a call: per sample what holds for all its rows (kHead words) and for each of its lists (kList tokens
// each, and one of biases) where each bucket begins (buckets + 1 numbers), then all samples' entries: a token's
// column in its bucket and its place, or with the top bit a bias's column and number.
constexpr int kHead = 8;
constexpr int kBucketBits = 11, kBucket = 1 << kBucketBits;
constexpr uint32_t kIsBias = 1u << 31;
constexpr int64_t kMaxBuckets = 8192;
constexpr int kTableThreads = 1024;
constexpr int kBiasSlots = 4096;
constexpr int64_t kList = 4096;
static_assert(2 * kBiasSlots <= kMaxBuckets && kMaxBias < kBiasSlots, "the biases' columns find a place");
static_assert(kBucket == kThreads * kG, "a slice is a whole number of buckets");
static_assert(kCountBits + kBucketBits <= 31, "an entry holds a token's place and column");

// kWide, kWideGrad: y, and its gradient, in fp32 whatever the logits' type (a filter reads them next).
enum Mode { kFwd, kBwd, kApply, kInPlace, kApplyGrad, kWide, kWideGrad };

struct Params {
  mirl_logit_processors A;
  const void* x;
  int64_t xsb, xsr;
  int64_t B, R, Rt, V;   // rows with a result; rows of the gradient (those past R: zeros)
  int64_t n_vocab;       // ids vs .. vs + n_vocab - 1 stand for the columns
  int64_t slices, chunks, buckets;
  int64_t lists;         // of a sample: of tokens, and one of biases if there are any
  const uint32_t* table;
  int rows;              // rows of a workgroup
  int32_t* left;         // kWide [B, R]: whether anything is left in a row
  void* y;               // processed logits, or a gradient
  int64_t ysb, ysr;
  const void* dy;        // kApplyGrad, kWideGrad
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

// The maximum and the sum over a wave within the VALU: each row of 16 lanes into its last, rows into the
// next, lanes 0 .. 31 into the others; the result in lane 63, given to all.  (A lane that nothing is
// permuted to keeps its own.  In asm: the compiler makes four instructions of a maximum's step; it knows
// nothing of the two wait states ahead of a permuted operand, hence the s_nops.)
__device__ __forceinline__ float wave_max_all(float v) {
  asm volatile(
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n\t"
      "s_nop 1"
      : "+v"(v));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
template <int CTRL>
__device__ __forceinline__ float from_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_sum_all(float v) {
  v += from_lane<0x111>(v);  // row_shr 1, 2, 4, 8
  v += from_lane<0x112>(v);
  v += from_lane<0x114>(v);
  v += from_lane<0x118>(v);
  v += from_lane<0x142>(v);  // row_bcast 15, 31
  v += from_lane<0x143>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float of_row(float v, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i)); }

// What holds for all rows of a sample, as the table's first words hold it.
struct Sample {
  float rp, inv_rp, pres, freq, inv_t;
  int n;       // tokens that row 0 follows
  int prompt;  // tokens of the prompt
  float t;     // the temperature
};
static_assert(sizeof(Sample) == kHead * 4, "the table's head");
__host__ __device__ __forceinline__ int64_t token_lists(int64_t n_ids) { return n_ids > kList ? (n_ids + kList - 1) / kList : 1; }
// Words of a sample ahead of all samples' entries.
__host__ __device__ __forceinline__ int64_t head_words(int64_t lists, int64_t buckets) { return kHead + lists * (buckets + 1); }
__device__ __forceinline__ const uint32_t* head_of(const Params& P, int64_t b) { return P.table + b * head_words(P.lists, P.buckets); }

// The bits of a where `mask` has them, else those of b.  (In asm: from the shifts and masks that follow, the
// compiler makes three instructions of it.)
__device__ __forceinline__ uint32_t either(uint32_t mask, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("v_bfi_b32 %0, %1, %2, %3" : "=v"(r) : "v"(mask), "s"(a), "v"(b));
  return r;
}

// v where bit e of `keep` is set, else `other`; as bits, whatever v holds.
__device__ __forceinline__ float keep_if(float v, uint32_t keep, int e, float other) {
  uint32_t t = (uint32_t)__builtin_amdgcn_sbfe((int)keep, e, 1);
  asm("" : "+v"(t));  // (two instructions, where a compare and a select take three)
  return __uint_as_float((__float_as_uint(v) & t) | (__float_as_uint(other) & ~t));
}

// z / d to the nearest, from inv = 1 / d to the nearest: the product is off by up to an ulp and a half, and its remainder, exact in
// one fma, gives the rest (P. Markstein, IBM J. Res. Dev. 34, 1990).  Infinities and NaN have no remainder and stay, and so does
// the sign of a zero (a remainder of 0 is +0, and is subtracted).  !EXACT: the
// product alone, where the result is rounded to 16 bits or goes into a logprob, whose sums are off by more.  (fp32 tokens written
// out 20.0 us either way.)
template <bool EXACT>
__device__ __forceinline__ float quotient(float z, float d, float inv) {
  const float q = z * inv;
  if constexpr (!EXACT) return q;
  const float r = fmaf(q, d, -z);
  return fabsf(r) < INFINITY ? fmaf(-r, inv, q) : q;
}

// Bias and penalties of one logit under its word.
template <bool EXACT>
__device__ __forceinline__ float penalized(float z, uint32_t w, const Sample& S, uint32_t& how) {
  how = 0;
  if (w & (kInPrompt | kCount)) {
    how = z > 0.f ? 1u : 256u;
    if constexpr (EXACT)
      z = z > 0.f ? quotient<true>(z, S.rp, S.inv_rp) : z * S.rp;
    else
      z *= z > 0.f ? S.inv_rp : S.rp;
  }
  const uint32_t n = w & kCount;
  z -= S.freq * (float)n;
  z -= n != 0 ? S.pres : 0.f;
  return z;
}

// Bias and penalties of a group's tokens: those of any lane of the wave (`any`, a scalar), in the
// lanes that have them (`bits`).  Returns which were divided by the repetition penalty (bits 0 .. 7) and
// which multiplied (8 .. 15).
template <bool EXACT, class F>
__device__ __forceinline__ uint32_t special(float (&v)[kG], uint32_t any, uint32_t bits, const vu4* words, F&& bias_of,
                                            const Sample& S) {
  uint32_t how = 0;
#pragma unroll
  for (int e = 0; e < kG; ++e) {
    if ((any & (1u << e)) == 0) continue;
    asm volatile("");  // (a branch of its own: the test of the lanes' bits is not worth making for nothing)
    if ((bits >> e) & 1u) {
      const uint32_t w = words[e / 4][e % 4];
      uint32_t h;
      v[e] = penalized<EXACT>(w >> kBiasShift ? v[e] + bias_of(w, e) : v[e], w, S, h);
      how |= h << e;
    }
  }
  return how;
}
// What the repetition penalty makes of a gradient.
__device__ __forceinline__ void through(float (&o)[kG], uint32_t any, uint32_t how, const Sample& S) {
#pragma unroll
  for (int e = 0; e < kG; ++e) {
    if ((any & (1u << e)) == 0) continue;
    asm volatile("");
    o[e] *= (how >> e) & 1u ? S.inv_rp : (how >> e) & 256u ? S.rp : 1.f;
  }
}

// Buckets of a list of one sample's tokens (those that any of the R rows follows), or of its biases.  An entry's place
// in its bucket comes from an atomic: the order differs from run to run, what is counted does not.  A workgroup
// has kList tokens, so that a long history is spread over the chip: one row of 151936 logits behind 131072 tokens,
// written out, takes 16 us where they are spread evenly and 56 where they follow Zipf's law (most in one slice, which
// one workgroup counts); with one workgroup for all of them 94 and 206.
// (And the flags that kWide's rows set, if there are any, begin as 0.)
__global__ __launch_bounds__(kTableThreads) void processors_table_kernel(mirl_logit_processors A, int64_t R, int64_t n_vocab,
                                                                         int64_t lists, int buckets, uint32_t* table, int32_t* left) {
  __shared__ uint32_t s_at[kMaxBuckets];
  __shared__ uint32_t s_wave[kTableThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t b = blockIdx.x / lists, list = blockIdx.x - b * lists, B = gridDim.x / lists;
  const bool biases = list == token_lists(A.n_ids);
  const int64_t* ids = A.ids + b * A.ids_stride_b;
  const int64_t* bias_ids = A.bias_ids + b * A.bias_stride_b;
  const int64_t n_b = min(A.lengths != nullptr ? A.lengths[b] : int64_t(1), A.n_ids);  // (what is beyond counts all tokens too)
  uint32_t* const head = table + b * head_words(lists, buckets);
  uint32_t* const begins = head + kHead + list * (buckets + 1);
  uint32_t* const entries = table + B * head_words(lists, buckets) + b * (A.n_ids + A.n_bias);
  if (list == 0 && tid == 0) {
    Sample S;
    S.rp = A.repetition != nullptr ? A.repetition[b] : A.repetition_all;
    S.inv_rp = 1.f / S.rp;
    S.pres = A.presence != nullptr ? A.presence[b] : A.presence_all;
    S.freq = A.frequency != nullptr ? A.frequency[b] : A.frequency_all;
    S.t = A.temperature != nullptr ? A.temperature[b] : A.temperature_all;
    S.inv_t = 1.f / S.t;
    S.n = (int)max(n_b, -(int64_t(1) << 30));
    S.prompt = A.prompt_lengths != nullptr ? (int)min(max(A.prompt_lengths[b], int64_t(0)), A.n_ids) : 0;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&S);
    for (int k = 0; k < kHead; ++k) head[k] = w[k];
  }
  if (left != nullptr && list == 0)
    for (int64_t r = tid; r < R; r += kTableThreads) left[b * R + r] = 0;
  auto column = [&](int64_t id) {
    const uint64_t c = (uint64_t)id - (uint64_t)A.vocab_start;
    return c < (uint64_t)n_vocab ? (int)c : -1;
  };
  // the list's tokens (place, column), or biases (number, column), of this thread
  constexpr int kOwn = kList / kTableThreads;
  static_assert(kList % kTableThreads == 0 && kMaxBias <= kList, "a thread holds its part of a list");
  const int64_t from = biases ? 0 : list * kList;
  const int n = biases ? (int)A.n_bias : (int)min(max(min(n_b + R - 1, A.n_ids) - from, int64_t(0)), kList);
  int own[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int k = i * kTableThreads + tid;
    own[i] = k < n ? column(biases ? bias_ids[k] : ids[(from + k) * A.ids_stride_s]) : -1;
  }
  // A bias holds if no later one of its sample names the same token: each column finds a slot of its own (open
  // addressing, at most half of the slots taken), which keeps the largest number that came by.
  if (biases && n > 1) {
    uint32_t* const s_column = s_at;
    uint32_t* const s_last = s_at + kBiasSlots;
    for (int k = tid; k < 2 * kBiasSlots; k += kTableThreads) s_at[k] = 0;
    __syncthreads();
    uint32_t slot[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (own[i] < 0) continue;
      uint32_t h = (uint32_t)own[i] * 0x9e3779b1u >> 20;
      for (;; h = (h + 1) % kBiasSlots) {
        const uint32_t was = atomicCAS(&s_column[h], 0u, (uint32_t)own[i] + 1);
        if (was == 0 || was == (uint32_t)own[i] + 1) break;
      }
      slot[i] = h;
      atomicMax(&s_last[h], (uint32_t)(i * kTableThreads + tid));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      if (own[i] >= 0 && s_last[slot[i]] != (uint32_t)(i * kTableThreads + tid)) own[i] = -1;
    __syncthreads();
  }
  for (int k = tid; k < buckets; k += kTableThreads) s_at[k] = 0;
  __syncthreads();
  // An atomic for each; its result is the entry's place in its bucket.
  uint32_t place[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i)
    if (own[i] >= 0) place[i] = atomicAdd(&s_at[own[i] >> kBucketBits], 1u);
  __syncthreads();
  // the sizes' running sum: a few buckets a thread, the threads' sums over waves and the workgroup
  const int per = (buckets + kTableThreads - 1) / kTableThreads, k0 = min(tid * per, buckets), k1 = min(k0 + per, buckets);
  uint32_t mine = 0;
  for (int k = k0; k < k1; ++k) mine += s_at[k];
  uint32_t upto = mine;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)upto, off, kWave);
    upto += lane >= off ? o : 0;
  }
  if (lane == kWave - 1) s_wave[wave] = upto;
  __syncthreads();
  uint32_t at = (uint32_t)(biases ? A.n_ids : from) + upto - mine;
  for (int w = 0; w < wave; ++w) at += s_wave[w];
  for (int k = k0; k < k1; ++k) {
    const uint32_t size = s_at[k];
    s_at[k] = at;
    begins[k] = at;
    at += size;
  }
  if (tid == kTableThreads - 1) begins[buckets] = at;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    if (own[i] >= 0)
      entries[s_at[own[i] >> kBucketBits] + place[i]] = (biases ? kIsBias : 0u) |
                                                        (uint32_t)(from + i * kTableThreads + tid) << kBucketBits |
                                                        (uint32_t)(own[i] & (kBucket - 1));
  }
}

// MASKED: there are grammar masks.
template <class E, int MODE, int NV, bool MASKED>
__global__ __launch_bounds__(kThreads) void processors_kernel(Params P) {
  using raw = typename E::raw;
  constexpr bool kWritten = MODE == kApply || MODE == kWide, kGradOfY = MODE == kApplyGrad || MODE == kWideGrad;
  using EY = std::conditional_t<MODE == kWide || MODE == kWideGrad, F32, E>;  // of y and its gradient
  using EI = std::conditional_t<kGradOfY, EY, E>;                             // of the values a row is read as: logits, or y's gradient
  using EO = std::conditional_t<MODE == kWide, F32, E>;                       // of what is written
  constexpr bool kExact = (kWritten || MODE == kInPlace) && std::is_same<EO, F32>::value;
  constexpr int kWaveCols = kWave * NV * kG, kSlice = kWaves * kWaveCols;
  constexpr int kPacks = (NV + 3) / 4;  // four groups' bytes in a word
  __shared__ __align__(16) uint32_t s_word[kSlice];
  // kFwd: up to 64 of a wave's tokens with a word are held by a lane each
  constexpr bool kLists = MODE == kFwd;
  __shared__ uint16_t s_list[kLists ? kWaves : 1][kWave];
  __shared__ __align__(16) raw s_row[kLists ? kSlice : 8];  // a row's values and mask bytes, for those lanes
  __shared__ uint8_t s_mask[kLists && MASKED ? kSlice / kG : 1];
  // kFwd: what a mask's byte (fp32: half of one) leaves of a 16-byte piece's words
  constexpr int kLut = kLists && MASKED ? 1 << E::kVec : 1;
  __shared__ vu4 s_lut[kLut];
  // the other modes: biases by column (a gather in the middle of a row would wait for the next row's loads)
  __shared__ float s_bias[kLists ? 1 : kSlice];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t slices = (uint32_t)P.slices, chunks = (uint32_t)P.chunks;
  // Neighbouring workgroups take neighbouring slices, from the first one on; where eight divides their number,
  // from another one in each run of rows: workgroups go to the eight dies in turn, and a die would always have
  // the same columns ([4, 1024, 131072] bf16 under masks, 32 slices: forward 229 us, without 301; the gradient of
  // written-out logits 435 and 483, of the logprobs, whose zero rows differ from run to run, 1.36 ms and 1.24).
  const uint32_t rest = blockIdx.x / slices;
  const uint32_t slice = (blockIdx.x + (MODE != kBwd && slices % 8 == 0 ? rest : 0)) % slices;
  const uint32_t chunk = rest % chunks, b = rest / chunks;
  const int64_t n0 = (int64_t)slice * kSlice;
  const int64_t r0 = (int64_t)chunk * P.rows;
  const int n_rows = (int)min((int64_t)P.rows, P.Rt - r0);
  const mirl_logit_processors& A = P.A;
  const uint32_t* head = head_of(P, b);
  const Sample S = *reinterpret_cast<const Sample*>(head);
  const int64_t* ids = A.ids + b * A.ids_stride_b;
  const float* bias = A.bias + b * A.bias_stride_b;

  const int g0 = wave * NV * kWave + lane;  // group u of the lane: g0 + 64 u
  const raw* xr = static_cast<const raw*>(P.x) + b * P.xsb + r0 * P.xsr + n0;
  const typename EY::raw* dyr = kGradOfY ? static_cast<const typename EY::raw*>(P.dy) + b * P.gsb + r0 * P.gsr + n0 : nullptr;
  typename EO::raw* yr = MODE == kFwd ? nullptr : static_cast<typename EO::raw*>(P.y) + b * P.ysb + r0 * P.ysr + n0;
  const uint32_t left = (uint32_t)min((int64_t)kSlice, P.V - n0);  // columns of the slice
  auto col = [&](int u) { return (uint32_t)(g0 + u * kWave) * kG; };
  const uint32_t at0 = g0 * kGroupBytes<E>;
  auto group_at = [&](auto t, int u) -> uint32_t {  // of t's elements, in bytes
    constexpr uint32_t bytes = kGroupBytes<decltype(t)>;
    if constexpr (bytes == kGroupBytes<E>)
      return at0 + u * kWave * bytes;
    else
      return (uint32_t)(g0 + u * kWave) * bytes;
  };
  auto put = [&](typename EO::raw* row, int u, const float (&v)[kG], bool whole) __attribute__((always_inline)) {
    if (whole || col(u) + kG <= left) {
      store_group<EO>(row, group_at(EO{}, u), v);
    } else {
#pragma unroll
      for (int e = 0; e < kG; ++e)
        if (col(u) + e < left) row[col(u) + e] = EO::from_float(v[e]);
    }
  };

  // What the rows need, row r0 + l in lane l.  kBwd: its gradient and statistics; rows without a gradient
  // are zeros and not read.
  uint64_t todo = n_rows == 64 ? ~0ull : (1ull << n_rows) - 1;
  float m_g = 0.f, m_M = 0.f, m_ls = 0.f;
  if constexpr (MODE == kBwd) {
    const int64_t r = r0 + lane;
    if (lane < n_rows && r < P.R) {
      m_g = P.g[b * P.gsb + r * P.gsr];
      m_M = P.stats[(b * P.R + r) * 2];
      m_ls = P.stats[(b * P.R + r) * 2 + 1];
      if (m_M == -INFINITY && m_ls == -INFINITY) m_g = 0.f;  // nothing was left in the row, or it has no next token
    }
    uint64_t zeros = todo;
    todo = __ballot(m_g != 0.f);
    zeros &= ~todo;
    const float z[kG] = {};
    for (; zeros != 0; zeros &= zeros - 1) {
      typename EO::raw* row = yr + __builtin_ctzll(zeros) * P.ysr;
#pragma unroll
      for (int u = 0; u < NV; ++u) put(row, u, z, false);
    }
    if (todo == 0) return;  // (the same in all waves)
  }
  // The first row's values are on their way while the tokens are counted.
  vu4 q[NV][kP<EI>];
  auto issue = [&](int i, int u, bool whole, uint32_t keep) __attribute__((always_inline)) {
    const typename EI::raw* row;
    if constexpr (kGradOfY)
      row = dyr + i * P.gsr;
    else
      row = xr + i * P.xsr;
    if (whole || col(u) + kG <= left) load_group<EI>(row, group_at(EI{}, u) & keep, q[u]);
  };
  const int first = __builtin_ctzll(todo);
  if constexpr (MODE != kInPlace) {
#pragma unroll
    for (int u = 0; u < NV; ++u) issue(first, u, false, ~0u);
  }

  // ---- the tokens ahead of row r0, and the biases ----
#pragma unroll
  for (int i = 0; i < kSlice / 4 / kThreads; ++i)
    reinterpret_cast<vu4*>(s_word)[i * kThreads + tid] = vu4{0u, 0u, 0u, 0u};
  if constexpr (kLists && MASKED) {
    if (tid < kLut) {
      vu4 w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (E::kVec == 8)
          w[k] = (tid >> (2 * k) & 1 ? 0xffffu : 0u) | (tid >> (2 * k + 1) & 1 ? 0xffff0000u : 0u);
        else
          w[k] = tid >> k & 1 ? ~0u : 0u;
      }
      s_lut[tid] = w;
    }
  }
  // an id's column in this wave, or -1
  const int64_t first_id = A.vocab_start + n0 + wave * kWaveCols;
  const uint32_t here = (uint32_t)max(int64_t(0), min((int64_t)kWaveCols, P.n_vocab - n0 - wave * kWaveCols));
  auto column = [&](int64_t id) {
    const uint64_t c = (uint64_t)id - (uint64_t)first_id;
    return c < here ? (int)c : -1;
  };
  const uint32_t buckets = (uint32_t)P.buckets, bucket0 = slice * NV, lists = (uint32_t)P.lists;
  const uint32_t* entries = P.table + P.B * head_words(P.lists, P.buckets) + b * (A.n_ids + A.n_bias);
  // where the slice's entries of a list begin, those of its second bucket, and where they end
  struct Span {
    uint32_t from, mid, to;
  };
  auto span_of = [&](uint32_t l) {
    const uint32_t* begins = head + kHead + (int64_t)l * (buckets + 1) + bucket0;
    const uint32_t mid = begins[1];
    return Span{begins[0], mid, NV > 1 ? begins[min(2u, buckets - bucket0)] : mid};
  };
  const bool few = lists <= 2;
  const Span first_span = few ? span_of(0) : Span{}, second_span = few && lists == 2 ? span_of(1) : Span{};
  const uint32_t ahead = (uint32_t)max(S.n + r0, int64_t(0)), in_prompt = (uint32_t)S.prompt;
  // The token that is new ahead of a row and the one behind it (columns of this wave, or -1), its mask.
  constexpr int kOfPrompt = 1 << 30;
  int m_new = -1, m_next = -1, m_mask = -1;
  if (lane < n_rows) {
    const int64_t r = r0 + lane, at = S.n + r;
    if (lane > 0 && at > 0 && at <= A.n_ids) {
      m_new = column(ids[(at - 1) * A.ids_stride_s]);
      if (m_new >= 0 && at - 1 < S.prompt) m_new |= kOfPrompt;
    }
    if constexpr (MODE == kFwd || MODE == kBwd) {
      if (at >= 0 && at < A.n_ids) m_next = column(ids[at * A.ids_stride_s]);
    }
    if (MASKED && (MODE != kBwd || r < P.R)) {
      const int64_t m = A.mask_rows[b * A.mask_rows_stride_b + r * A.mask_rows_stride_r];
      m_mask = m >= 0 && m < A.n_masks ? (int)m : -1;
    }
  }
  // entry w, number i of the table; from `mid` on a list's entries are those of the second bucket
  auto count = [&](uint32_t w, uint32_t i, uint32_t mid) __attribute__((always_inline)) {
    const uint32_t at = (w & ~kIsBias) >> kBucketBits;
    const uint32_t c = (w & (kBucket - 1)) + (NV > 1 && i >= mid ? kBucket : 0);
    if (w & kIsBias) {
      atomicAdd(&s_word[c], (at + 1) << kBiasShift);
      if constexpr (!kLists) s_bias[c] = bias[at];
    } else if (at < ahead && at < in_prompt) {
      atomicOr(&s_word[c], kInPrompt);
    } else if (at < ahead) {
      atomicAdd(&s_word[c], 1u);
    }
  };
  __syncthreads();
  bool some = false;
  // Loads under way at a time (one row behind 8192 tokens, of which one slice has most: 14.5 us with four for a
  // thread, 16.6 with one; behind 131072 with eight 56, with four 65).
  constexpr int kFew = 4, kMany = 8;
  if (few) {  // one after the other; what leads to them is loaded by scalars, ahead of all this
    const uint32_t n = first_span.to - first_span.from, all = n + second_span.to - second_span.from;
    some = all != 0;
    auto place = [&](uint32_t k) { return k + (k < n ? first_span.from : second_span.from - n); };
    for (uint32_t k0 = 0; k0 < all; k0 += kFew * kThreads) {
      uint32_t w[kFew];
#pragma unroll
      for (int d = 0; d < kFew; ++d) w[d] = entries[place(min(k0 + d * kThreads + tid, all - 1))];
#pragma unroll
      for (int d = 0; d < kFew; ++d) {
        const uint32_t k = k0 + d * kThreads + tid;
        if (k < all) count(w[d], place(k), k < n ? first_span.mid : second_span.mid);
      }
    }
  } else {  // each wave a list, those behind the first row left out
    for (uint32_t l0 = 0; l0 < lists; l0 += kWave) {
      const uint32_t l = l0 + lane, n_lists = min(lists - l0, (uint32_t)kWave);
      Span at{};
      if (l < lists && (l * kList < ahead || l == (uint32_t)token_lists(A.n_ids))) at = span_of(l);
      some |= __ballot(at.from != at.to) != 0;
      for (uint32_t k = wave; k < n_lists; k += kWaves) {
        const uint32_t k_from = __builtin_amdgcn_readlane(at.from, k), k_mid = __builtin_amdgcn_readlane(at.mid, k),
                       k_to = __builtin_amdgcn_readlane(at.to, k);
        for (uint32_t i = k_from; i < k_to; i += kMany * kWave) {
          uint32_t w[kMany];
#pragma unroll
          for (int d = 0; d < kMany; ++d) w[d] = entries[min(i + d * kWave + lane, k_to - 1)];
#pragma unroll
          for (int d = 0; d < kMany; ++d)
            if (i + d * kWave + lane < k_to) count(w[d], i + d * kWave + lane, k_mid);
        }
      }
    }
  }
  const uint64_t new_rows = __ballot(m_new >= 0);
  __syncthreads();

  // ---- from here on each wave by itself ----
  const vu4* words = reinterpret_cast<const vu4*>(s_word) + g0 * (kG / 4);
  constexpr int kU = kWave * (kG / 4);  // between the lane's groups
  auto bias_of = [&](uint32_t w, int u, int e) { return kLists ? bias[(w >> kBiasShift) - 1] : s_bias[kLists ? 0 : col(u) + e]; };
  // Tokens with a word other than 0: a byte per group of the lane's and of any lane's.
  uint32_t bits[kPacks] = {}, any[kPacks] = {};
  // kFwd: the listed tokens (column, word, bias of the lane's), which are formed all at once and left out
  // of the groups (`gone` masks the lane's in the words of a group as it is read); the others as in every mode.
  constexpr int kRawWords = kLists ? kP<E> * 4 : 1, kPerWord = kG / (kP<E> * 4);
  uint32_t gone[kLists ? NV : 1][kRawWords] = {};
  auto mark_gone = [&](int u, int e) __attribute__((always_inline)) {  // (u and e constant)
    if constexpr (kLists) gone[u][e / kPerWord] |= kPerWord == 1 ? ~0u : 0xffffu << (16 * (e % kPerWord));
  };
  int listed = 0, h_col = -1;
  uint32_t h_word = 0;
  float h_bias = 0.f;
  if (some) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const vu4 lo = words[u * kU], hi = words[u * kU + 1];
#pragma unroll
      for (int e = 0; e < kG; ++e) {
        const bool set = (e < 4 ? lo[e & 3] : hi[e & 3]) != 0;
        const uint64_t all = __ballot(set);
        if (all == 0) continue;
        const uint32_t bit = 1u << (8 * (u % 4) + e);
        bool in_list = false;
        if constexpr (kLists) {
          const int at = listed + (int)__popcll(all & ((1ull << lane) - 1));
          in_list = set && at < kWave;
          if (in_list) s_list[wave][at] = (uint16_t)((u * kWave + lane) * kG + e);
          const int n = (int)__popcll(all);
          if (in_list) mark_gone(u, e);
          if (listed + n > kWave) any[u / 4] |= bit;
          listed = min(listed + n, kWave);
        } else {
          any[u / 4] |= bit;
        }
        if (set && !in_list) bits[u / 4] |= bit;
      }
    }
    if constexpr (kLists) {
      __builtin_amdgcn_wave_barrier();
      if (lane < listed) {
        h_col = s_list[wave][lane];
        h_word = s_word[wave * kWaveCols + h_col];
        if (h_word >> kBiasShift) h_bias = bias[(h_word >> kBiasShift) - 1];
      }
    }
  }
  // the token that is new ahead of row i
  auto add_token = [&](int i) __attribute__((always_inline)) {
    const int t = __builtin_amdgcn_readlane(m_new, i);
    const int c = t & (kOfPrompt - 1), group = c / kG;
    const uint32_t bit = 1u << (c % kG);
    auto more_of = [&](uint32_t w) { return t & kOfPrompt ? w | kInPrompt : w + 1; };
    const bool mine = group % kWave == lane;
    bool lists = false;
    if constexpr (kLists) {
      const bool held = h_col == c;
      if (__ballot(held) != 0) {
        if (held) h_word = more_of(h_word);
        return;
      }
      bool counted = false;  // one that is not listed
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (group / kWave == u) counted = __ballot(mine && ((bits[u / 4] >> (8 * (u % 4))) & bit)) != 0;
      lists = !counted && listed < kWave;
      if (lists) {
        if (lane == listed) {
          h_col = c;
          h_word = more_of(0);
        }
        ++listed;
      }
    }
    if (lists) {
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < kG; ++e)
          if (mine && group / kWave == u && c % kG == e) mark_gone(u, e);
      return;
    }
    if (mine) {
      uint32_t& w = s_word[wave * kWaveCols + c];
      w = more_of(w);
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (group / kWave != u) continue;
      const uint32_t b8 = bit << (8 * (u % 4));
      any[u / 4] |= b8;
      if (mine) bits[u / 4] |= b8;
    }
  };
  auto add_tokens = [&](int from, int to) __attribute__((always_inline)) {  // ahead of rows from + 1 .. to
    uint64_t some = new_rows & (~0ull << from << 1) & (~0ull >> (63 - to));
    for (; some != 0; some &= some - 1) add_token(__builtin_ctzll(some));
  };
  add_tokens(0, first);
  auto wave_bits = [&](int u) { return (any[u / 4] >> (8 * (u % 4))) & 0xffu; };
  auto lane_bits = [&](int u) { return (bits[u / 4] >> (8 * (u % 4))) & 0xffu; };

  // WHOLE: the slice lies inside the row.  Its loads are then issued in every row alike (behind the last
  // one, and in lanes that need nothing, of the slice's first columns): the compiler counts what is in flight,
  // and a row waits for its own values only.
  auto rows = [&](auto whole_c) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole_c)::value;
    auto tail = [&](auto et, const auto* row, int u, float fill, float (&v)[kG]) {
#pragma unroll
      for (int e = 0; e < kG; ++e) v[e] = col(u) + e < left ? decltype(et)::load(row + col(u) + e) : fill;
    };
    auto full = [&](int u) { return WHOLE || col(u) + kG <= left; };
    // a row's mask bytes; with y's gradient, the logits of groups with a word (as they come: what converts them would
    // wait here)
    uint8_t mk[NV];
    vu4 qx[kGradOfY ? NV : 1][kP<E>];
    auto mask_of = [&](int i) {
      const int m = __builtin_amdgcn_readlane(m_mask, i);
      return reinterpret_cast<const uint8_t*>(A.masks + (int64_t)max(m, 0) * A.mask_stride) + n0 / kG;
    };
    auto issue_mask = [&](int i, int u) __attribute__((always_inline)) {
      if constexpr (MASKED) {
        if (WHOLE || col(u) < left) mk[u] = mask_of(i)[g0 + u * kWave];
      }
    };
    auto issue_words = [&](int i) __attribute__((always_inline)) {
      if constexpr (kGradOfY) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
          if (full(u)) load_group<E>(xr + i * P.xsr, lane_bits(u) != 0 ? group_at(E{}, u) : 0, qx[u]);
      }
    };
#pragma unroll
    for (int u = 0; u < NV; ++u) issue_mask(first, u);
    issue_words(first);

    for (int i = first;;) {
      todo &= todo - 1;
      const bool more = todo != 0;
      const int next = more ? __builtin_ctzll(todo) : i;
      const bool masked = MASKED && __builtin_amdgcn_readlane(m_mask, i) >= 0;
      const typename EI::raw* row;
      if constexpr (kGradOfY)
        row = dyr + i * P.gsr;
      else
        row = xr + i * P.xsr;
      typename EO::raw* y_row = MODE == kFwd ? nullptr : yr + i * P.ysr;
      uint32_t allowed[NV];
      // group u of this row, and the next row's on its way
      auto take = [&](int u, float fill, float (&v)[kG]) __attribute__((always_inline)) {
        if (full(u)) {
          if constexpr (kLists) {
            if (listed > 0) {
#pragma unroll
              for (int k = 0; k < kP<E>; ++k) reinterpret_cast<vu4*>(s_row + col(u))[k] = q[u][k];
            }
            // (a masked token's bias and penalties leave it at -inf)
#pragma unroll
            for (int k = 0; k < kP<E>; ++k) {
              vu4 left_out = {gone[u][4 * k], gone[u][4 * k + 1], gone[u][4 * k + 2], gone[u][4 * k + 3]};
              if (masked) left_out |= ~s_lut[mk[u] >> (k * E::kVec) & (kLut - 1)];
#pragma unroll
              for (int j = 0; j < 4; ++j) q[u][k][j] = either(left_out[j], E::kNegInf2, q[u][k][j]);
            }
          }
          unpack_group<EI>(q[u], v);
        } else {
          tail(EI{}, row, u, fill, v);
          if constexpr (kLists) {
#pragma unroll
            for (int e = 0; e < kG; ++e) s_row[col(u) + e] = E::from_float(v[e]);  // (exact)
#pragma unroll
            for (int e = 0; e < kG; ++e)
              v[e] = (gone[u][e / kPerWord] >> (kPerWord == 1 ? 0 : 16 * (e % kPerWord)) & 1u) ||
                             (masked && !(mk[u] >> e & 1))
                         ? -INFINITY
                         : v[e];
          }
        }
        allowed[u] = masked ? mk[u] : 0xffu;
        if (kLists && masked && listed > 0) s_mask[kLists && MASKED ? g0 + u * kWave : 0] = (uint8_t)allowed[u];
        issue(next, u, WHOLE, more ? ~0u : 0u);
        issue_mask(next, u);
      };
      // the next token's group of the lane, and which of its eight
      int t = -1, tu = -1, tlane = -1, te = -1;
      if constexpr (MODE == kFwd || MODE == kBwd) {
        t = __builtin_amdgcn_readlane(m_next, i);
        if (t >= 0) {
          tu = t / (kG * kWave);
          tlane = t / kG % kWave;
          te = t % kG;
        }
      }
      if constexpr (MODE == kFwd) {
        float v[NV][kG];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          take(u, -INFINITY, v[u]);
          if (wave_bits(u) != 0)  // (a masked token's bias must not meet the -inf that the mask left)
            special<kExact>(v[u], wave_bits(u), lane_bits(u) & allowed[u], words + u * kU, [&](uint32_t w, int e) { return bias_of(w, u, e); }, S);
#pragma unroll
          for (int e = 0; e < kG; ++e) mx = fmaxf(mx, v[u][e]);
        }
        float h_y = -INFINITY;
        if (listed > 0) {
          uint32_t how;
          const int c = wave * kWaveCols + max(h_col, 0);
          h_y = penalized<false>(E::load(s_row + (kLists ? c : 0)) + h_bias, h_word, S, how);
          const uint32_t m = masked ? s_mask[kLists && MASKED ? c / kG : 0] : 0xffu;
          h_y = h_col >= 0 && (m >> (c % kG) & 1u) ? h_y : -INFINITY;
          mx = fmaxf(mx, h_y);
        }
        if (t >= 0) {
          const bool held = h_col == t;
          float xt = h_y;
          if (__ballot(held) == 0) {
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
              for (int e = 0; e < kG; ++e) xt = u == tu && e == te ? v[u][e] : xt;
          }
          if (__ballot(held) != 0 ? held : lane == tlane) P.xt[b * P.R + r0 + i] = xt;
        }
        // sums of 2^(y c - fl(M c)) with c = log2(e) / T, M the wave's maximum
        const float c = kLog2e * S.inv_t;
        const float M = wave_max_all(mx);
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
        if (listed > 0) {
          // (a lane without one: 2^-inf, or nothing under a maximum that is not there)
          s4[0] += in_range ? fast_exp2(fmaf(h_y, c, -off)) : M != -INFINITY ? fast_exp2((h_y - M) * c) : h_y != h_y ? h_y : 0.f;
        }
        float s = wave_sum_all((s4[0] + s4[1]) + (s4[2] + s4[3]));
        if (in_range) s *= fast_exp2(-fmaf(M, c, -off));  // the offset's rounding undone
        if (lane == 0)
          reinterpret_cast<float2*>(P.part)[(b * P.R + r0 + i) * (P.slices * kWaves) + slice * kWaves + wave] = float2{M, s};
      } else if constexpr (MODE == kBwd) {
        const float M = of_row(m_M, i), c = kLog2e * S.inv_t, ls = of_row(m_ls, i) * kLog2e, gt = of_row(m_g, i) * S.inv_t;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          float v[kG], o[kG];
          take(u, 0.f, v);
          uint32_t how = 0;
          if (wave_bits(u) != 0)
            how = special<kExact>(v, wave_bits(u), lane_bits(u), words + u * kU, [&](uint32_t w, int e) { return bias_of(w, u, e); }, S);
#pragma unroll
          for (int e = 0; e < kG; ++e) o[e] = fast_exp2(fmaf(v[e] - M, c, -ls)) * -gt;
          if (u == tu) {
#pragma unroll
            for (int e = 0; e < kG; ++e)
              o[e] = lane == tlane && e == te ? (1.f - fast_exp2(fmaf(v[e] - M, c, -ls))) * gt : o[e];
          }
          if (wave_bits(u) != 0) through(o, wave_bits(u), how, S);
          if (masked) {
#pragma unroll
            for (int e = 0; e < kG; ++e) o[e] = keep_if(o[e], allowed[u], e, 0.f);
          }
          put(y_row, u, o, WHOLE);
        }
      } else if constexpr (kWritten) {
        bool some_left = false;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          float v[kG];
          take(u, 0.f, v);
          if (wave_bits(u) != 0)
            special<kExact>(v, wave_bits(u), lane_bits(u), words + u * kU, [&](uint32_t w, int e) { return bias_of(w, u, e); }, S);
#pragma unroll
          for (int e = 0; e < kG; ++e) v[e] = quotient<kExact>(v[e], S.t, S.inv_t);
          if (masked) {
#pragma unroll
            for (int e = 0; e < kG; ++e) v[e] = keep_if(v[e], allowed[u], e, -INFINITY);
          }
          if constexpr (MODE == kWide) {
#pragma unroll
            for (int e = 0; e < kG; ++e) some_left |= v[e] != -INFINITY && (WHOLE || col(u) + e < left);
          }
          put(y_row, u, v, WHOLE);
        }
        if constexpr (MODE == kWide) {  // (any wave of any workgroup: all write the same)
          if (__ballot(some_left) != 0 && lane == 0) P.left[b * P.R + r0 + i] = 1;
        }
      } else if constexpr (kGradOfY) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          float v[kG];
          take(u, 0.f, v);
#pragma unroll
          for (int e = 0; e < kG; ++e) v[e] *= S.inv_t;
          if (wave_bits(u) != 0) {
            float x[kG];
            if (full(u))
              unpack_group<E>(qx[u], x);
            else
              tail(E{}, xr + i * P.xsr, u, 0.f, x);
            const uint32_t how =
                special<kExact>(x, wave_bits(u), lane_bits(u), words + u * kU, [&](uint32_t w, int e) { return bias_of(w, u, e); }, S);
            through(v, wave_bits(u), how, S);
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < kG; ++e) v[e] = keep_if(v[e], allowed[u], e, 0.f);
          }
          put(y_row, u, v, WHOLE);
        }
      } else {  // kInPlace: what changes
        const bool dense = S.t != 1.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          allowed[u] = masked ? mk[u] : 0xffu;
          issue_mask(next, u);
          if (!(WHOLE || col(u) < left) || !(dense || lane_bits(u) != 0 || allowed[u] != 0xffu)) continue;
          float v[kG];
          if (full(u)) {
            vu4 w[kP<E>];
            load_group<E>(row, group_at(E{}, u), w);
            unpack_group<E>(w, v);
          } else {
            tail(E{}, row, u, 0.f, v);
          }
          special<kExact>(v, wave_bits(u), lane_bits(u), words + u * kU, [&](uint32_t w, int e) { return bias_of(w, u, e); }, S);
#pragma unroll
          for (int e = 0; e < kG; ++e) v[e] = keep_if(quotient<kExact>(v[e], S.t, S.inv_t), allowed[u], e, -INFINITY);
          put(y_row, u, v, WHOLE);
        }
      }
      if (more) add_tokens(i, next);  // (this row is done with the words)
      issue_words(next);
      if (!more) break;
      i = next;
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
  const Sample S = *reinterpret_cast<const Sample*>(head_of(P, b));
  const float inv_t = S.inv_t, c = kLog2e * inv_t;
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
  const int64_t at = S.n + r;
  const int64_t t = at >= 0 && at < A.n_ids ? A.ids[b * A.ids_stride_b + at * A.ids_stride_s] - A.vocab_start : -1;
  const float logsum = logf(s);
  const bool scored = t >= 0 && t < P.n_vocab;
  out[row] = !scored ? 0.f : M == -INFINITY && s == 0.f ? -INFINITY : (P.xt[row] - M) * inv_t - logsum;
  if (stats != nullptr) {  // (a constant 0 has no gradient, as a row in which nothing is left)
    stats[2 * row] = scored ? M : -INFINITY;
    stats[2 * row + 1] = scored ? logsum : -INFINITY;
  }
}

// Rows of kWide in which nothing is left become a finite ramp, which any filter cuts as ordinary logits (of a row of -inf it
// forms (-inf) - (-inf)); what it makes of them is not used.
__global__ __launch_bounds__(kThreads) void processors_ramp_kernel(Params P) {
  const float step = -256.f / (float)P.V;
  for (int64_t row = blockIdx.x; row < P.B * P.R; row += gridDim.x) {
    if (P.left[row] != 0) continue;
    float* y = static_cast<float*>(P.y) + row / P.R * P.ysb + row % P.R * P.ysr;
    for (int64_t j = threadIdx.x; j < P.V; j += kThreads) y[j] = step * (float)j;
  }
}
constexpr int64_t kRampGrid = 4096;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Groups of a lane and rows of a workgroup.  The forward of 16-bit rows takes two groups (16 bytes each) where there
// are workgroups enough ([8, 2048, 151936] bf16, 16 rows, at an early stage: 1174 us, with one 1420, with four 1281;
// with 32 rows now 929 and 1006 with four), one where there are not; fp32 one of 32 bytes ([3, 256, 32003], 8 rows:
// 24 us, with two 26).  The others take one: narrow slices keep what is read and written close together (backward of
// the large rows 1.41 ms with one, 1.53 with two).  In the forward many rows share the count of the tokens ahead of
// them (929 us with 32, 959 with 16); where rows are written, few at a time reach across less memory: written out
// [2, 2048, 151936] 412 us with 4, 446 with 8, 465 with 2; the backward 1.36 ms with 4, 1.39 with 8, 1.57 with 2.  Fewer
// rows where there would be less than some rounds of workgroups (the fp32 forward 24 us with 8, 29 with 16, 44 with
// 32; its backward 41 with 4, 45 with 8).
struct Plan {
  int nv;
  int64_t slices, rows, chunks;
};
Plan plan_of(int mode, int dtype, int64_t B, int64_t R, int64_t V) {
  Plan p;
  const int64_t wide = ceil_div(V, kBucket);
  p.nv = mode == kFwd && dtype != MIRL_DTYPE_F32 && B * R * wide >= 4096 ? 2 : 1;
  p.slices = ceil_div(V, kBucket * p.nv);
  p.rows = mode == kFwd ? 32 : 4;
  auto workgroups = [&] { return B * ceil_div(R, p.rows) * p.slices; };
  while (p.rows > 8 && workgroups() < 8192) p.rows /= 2;
  while (p.rows > 1 && workgroups() < (mode == kFwd ? 1024 : 2048)) p.rows /= 2;
  while (workgroups() >= (int64_t(1) << 24) && p.rows < kWave) p.rows *= 2;
  p.chunks = ceil_div(R, p.rows);
  return p;
}

int make_table(const Params& P, int64_t rows, uint32_t* table, const char* what, hipStream_t st) {
  hipLaunchKernelGGL(processors_table_kernel, dim3((unsigned)(P.B * P.lists)), dim3(kTableThreads), 0, st, P.A, rows, P.n_vocab,
                     P.lists, (int)P.buckets, table, P.left);
  return check_launch(what);
}

// `table`: the one to make ahead of the rows (a backward has its forward's).
template <int MODE>
int launch(Params& P, int dtype, int64_t rows, const char* what, hipStream_t st, uint32_t* table = nullptr) {
  const Plan p = plan_of(MODE, dtype, P.B, rows, P.V);
  P.slices = p.slices;
  P.chunks = p.chunks;
  P.rows = (int)p.rows;
  MIRL_REQUIRE(P.B * p.chunks * p.slices < (int64_t(1) << 24), "too many rows of %lld columns", (long long)P.V);
  if (table != nullptr)
    if (int e = make_table(P, rows, table, what, st)) return e;
  const dim3 grid((unsigned)(P.B * p.chunks * p.slices)), block(kThreads);
  auto go = [&](auto e, auto nv, auto masked) {
    hipLaunchKernelGGL((processors_kernel<decltype(e), MODE, decltype(nv)::value, decltype(masked)::value>), grid, block, 0, st, P);
  };
  auto go_masked = [&](auto e, auto nv) {
    if (P.A.n_masks > 0)
      go(e, nv, std::true_type{});
    else
      go(e, nv, std::false_type{});
  };
  auto go_type = [&](auto e) {
    if constexpr (MODE == kFwd) {
      if constexpr (!std::is_same<decltype(e), F32>::value) {
        if (p.nv == 2) return go_masked(e, std::integral_constant<int, 2>{});
      }
    }
    go_masked(e, std::integral_constant<int, 1>{});
  };
  if (dtype == MIRL_DTYPE_F32)
    go_type(F32{});
  else if (dtype == MIRL_DTYPE_BF16)
    go_type(BF16{});
  else
    go_type(F16{});
  return check_launch(what);
}

int check_args(const mirl_logit_processors* A, int dtype, int64_t B, int64_t R, int64_t V) {
  MIRL_REQUIRE(dtype == MIRL_DTYPE_F32 || dtype == MIRL_DTYPE_BF16 || dtype == MIRL_DTYPE_F16,
               "unsupported logits dtype code %d", dtype);
  MIRL_REQUIRE(A != nullptr, "null pointer argument");
  MIRL_REQUIRE(B >= 0 && R >= 0 && V > 0, "invalid shape B=%lld R=%lld V=%lld", (long long)B, (long long)R, (long long)V);
  MIRL_REQUIRE(V <= kMaxBuckets * kBucket, "a vocabulary of %lld exceeds %lld", (long long)V, (long long)(kMaxBuckets * kBucket));
  MIRL_REQUIRE(B < (int64_t(1) << 31) && R < (int64_t(1) << 31) && B * R < (int64_t(1) << 31), "sizes exceed 2^31-1");
  MIRL_REQUIRE(A->n_ids >= 0 && A->n_ids <= kMaxTokens, "%lld tokens of a sample, at most %lld are counted",
               (long long)A->n_ids, (long long)kMaxTokens);
  MIRL_REQUIRE(A->n_bias >= 0 && A->n_bias <= kMaxBias, "%lld biases of a sample, at most %lld are held",
               (long long)A->n_bias, (long long)kMaxBias);
  MIRL_REQUIRE(A->n_masks >= 0 && (A->n_masks == 0 || A->mask_stride >= ceil_div(V, 32)),
               "grammar masks of %lld words do not cover %lld columns", (long long)A->mask_stride, (long long)V);
  // a launch holds fewer than 2^32 threads; the table takes 1024 for each list
  const int64_t lists = token_lists(A->n_ids) + (A->n_bias > 0);
  MIRL_REQUIRE(B * lists < (int64_t(1) << 22), "too many samples (%lld) with %lld lists of tokens and biases each", (long long)B, (long long)lists);
  if (B * R == 0) return MIRL_OK;
  MIRL_REQUIRE((A->n_ids == 0 || A->ids != nullptr) && (A->n_bias == 0 || (A->bias_ids != nullptr && A->bias != nullptr)) &&
                   (A->n_masks == 0 || (A->masks != nullptr && A->mask_rows != nullptr)),
               "null pointer argument");
  return MIRL_OK;
}

Params params_of(const mirl_logit_processors* A, const uint32_t* table, const void* x, int64_t B, int64_t R, int64_t Rt, int64_t V, int64_t xsb,
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
  P.n_vocab = n < 0 ? 0 : n < V ? n : V;
  P.buckets = ceil_div(V, kBucket);
  P.lists = token_lists(A->n_ids) + (A->n_bias > 0);
  P.table = table;
  return P;
}

}  // namespace
}  // namespace mirl

using namespace mirl;

extern "C" int64_t mirl_logit_processors_table_elems(int64_t B, int64_t V, int64_t n_ids, int64_t n_bias) {
  if (B <= 0 || V <= 0 || n_ids < 0 || n_bias < 0) return 0;
  return B * (head_words(token_lists(n_ids) + (n_bias > 0), ceil_div(V, kBucket)) + n_ids + n_bias);
}

extern "C" int64_t mirl_processed_logprob_workspace_elems(int64_t B, int64_t R, int64_t V) {
  if (B <= 0 || R <= 0 || V <= 0) return 0;
  return B * R * (plan_of(kFwd, MIRL_DTYPE_F32, B, R, V).slices * kWaves * 2 + 1);
}

extern "C" int mirl_processed_logprob_fwd(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                          int64_t stride_r, const mirl_logit_processors* processors, uint32_t* table, float* out,
                                          float* stats, float* workspace, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, R, V)) return e;
  if (B * R == 0) return MIRL_OK;
  // (a wave joins a row's parts, and a launch holds fewer than 2^32 threads)
  MIRL_REQUIRE(B * R < (int64_t(1) << 26), "%lld rows: fewer than 2^26 are scored in a call", (long long)(B * R));
  MIRL_REQUIRE(table && logits && out && workspace, "null pointer argument");
  Params P = params_of(processors, table, logits, B, R, R, V, stride_b, stride_r);
  hipStream_t st = static_cast<hipStream_t>(stream);
  P.part = workspace;
  P.xt = workspace + B * R * plan_of(kFwd, dtype, B, R, V).slices * kWaves * 2;
  if (int e = launch<kFwd>(P, dtype, R, "mirl_processed_logprob_fwd", st, table)) return e;
  hipLaunchKernelGGL(processors_join_kernel, dim3((unsigned)ceil_div(B * R, kWaves)), dim3(kThreads), 0, st, P, out, stats);
  return check_launch("mirl_processed_logprob_fwd");
}

extern "C" int mirl_processed_logprob_bwd(const void* logits, int dtype, int64_t B, int64_t R, int64_t Rt, int64_t V,
                                          int64_t stride_b, int64_t stride_r, const mirl_logit_processors* processors, const uint32_t* table,
                                          const float* stats, const float* grad_out, int64_t g_stride_b, int64_t g_stride_r,
                                          void* grad_in, int64_t gi_stride_b, int64_t gi_stride_r, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, Rt, V)) return e;
  MIRL_REQUIRE(R >= 0 && R <= Rt, "invalid shape R=%lld of %lld rows", (long long)R, (long long)Rt);
  if (B * Rt == 0) return MIRL_OK;
  MIRL_REQUIRE(table && logits && grad_in && (R == 0 || (stats && grad_out)), "null pointer argument");
  Params P = params_of(processors, table, logits, B, R, Rt, V, stride_b, stride_r);
  P.stats = stats;
  P.g = grad_out;
  P.gsb = g_stride_b;
  P.gsr = g_stride_r;
  P.y = grad_in;
  P.ysb = gi_stride_b;
  P.ysr = gi_stride_r;
  return launch<kBwd>(P, dtype, Rt, "mirl_processed_logprob_bwd", static_cast<hipStream_t>(stream));
}

namespace mirl {
namespace {
// MODE: kApply (which becomes kInPlace where out is the logits) or kWide.
template <int MODE>
int write_processed(const char* what, const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b, int64_t stride_r,
                    const mirl_logit_processors* processors, uint32_t* table, void* out, int64_t o_stride_b, int64_t o_stride_r,
                    int32_t* left, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, R, V)) return e;
  if (B * R == 0) return MIRL_OK;
  MIRL_REQUIRE(table && logits && out && (MODE == kApply || left), "null pointer argument");
  MIRL_REQUIRE(MODE == kApply ? out != logits || (o_stride_b == stride_b && o_stride_r == stride_r) : out != logits,
               MODE == kApply ? "in place, the strides are those of the logits" : "fp32 values are not written in place");
  Params P = params_of(processors, table, logits, B, R, R, V, stride_b, stride_r);
  P.y = out;
  P.ysb = o_stride_b;
  P.ysr = o_stride_r;
  P.left = left;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if constexpr (MODE == kApply) {
    return out == logits ? launch<kInPlace>(P, dtype, R, what, st, table) : launch<kApply>(P, dtype, R, what, st, table);
  } else {
    if (int e = launch<kWide>(P, dtype, R, what, st, table)) return e;
    hipLaunchKernelGGL(processors_ramp_kernel, dim3((unsigned)(B * R < kRampGrid ? B * R : kRampGrid)), dim3(kThreads), 0, st, P);
    return check_launch(what);
  }
}

template <int MODE>
int write_gradient(const char* what, const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b, int64_t stride_r,
                   const mirl_logit_processors* processors, const uint32_t* table, const void* grad_out, int64_t g_stride_b,
                   int64_t g_stride_r, void* grad_in, int64_t gi_stride_b, int64_t gi_stride_r, void* stream) {
  clear_error();
  if (int e = check_args(processors, dtype, B, R, V)) return e;
  if (B * R == 0) return MIRL_OK;
  MIRL_REQUIRE(table && logits && grad_out && grad_in, "null pointer argument");
  Params P = params_of(processors, table, logits, B, R, R, V, stride_b, stride_r);
  P.dy = grad_out;
  P.gsb = g_stride_b;
  P.gsr = g_stride_r;
  P.y = grad_in;
  P.ysb = gi_stride_b;
  P.ysr = gi_stride_r;
  return launch<MODE>(P, dtype, R, what, static_cast<hipStream_t>(stream));
}
}  // namespace
}  // namespace mirl

extern "C" int mirl_process_logits(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                   int64_t stride_r, const mirl_logit_processors* processors, uint32_t* table, void* out,
                                   int64_t o_stride_b, int64_t o_stride_r, void* stream) {
  return write_processed<kApply>("mirl_process_logits", logits, dtype, B, R, V, stride_b, stride_r, processors, table, out,
                                 o_stride_b, o_stride_r, nullptr, stream);
}

extern "C" int mirl_process_logits_bwd(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                       int64_t stride_r, const mirl_logit_processors* processors, const uint32_t* table, const void* grad_out,
                                       int64_t g_stride_b, int64_t g_stride_r, void* grad_in, int64_t gi_stride_b,
                                       int64_t gi_stride_r, void* stream) {
  return write_gradient<kApplyGrad>("mirl_process_logits_bwd", logits, dtype, B, R, V, stride_b, stride_r, processors, table, grad_out,
                                    g_stride_b, g_stride_r, grad_in, gi_stride_b, gi_stride_r, stream);
}

extern "C" int mirl_process_logits_f32(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                       int64_t stride_r, const mirl_logit_processors* processors, uint32_t* table, float* out,
                                       int64_t o_stride_b, int64_t o_stride_r, int32_t* left, void* stream) {
  return write_processed<kWide>("mirl_process_logits_f32", logits, dtype, B, R, V, stride_b, stride_r, processors, table, out,
                                o_stride_b, o_stride_r, left, stream);
}

extern "C" int mirl_process_logits_f32_bwd(const void* logits, int dtype, int64_t B, int64_t R, int64_t V, int64_t stride_b,
                                           int64_t stride_r, const mirl_logit_processors* processors, const uint32_t* table,
                                           const float* grad_out, int64_t g_stride_b, int64_t g_stride_r, void* grad_in,
                                           int64_t gi_stride_b, int64_t gi_stride_r, void* stream) {
  return write_gradient<kWideGrad>("mirl_process_logits_f32_bwd", logits, dtype, B, R, V, stride_b, stride_r, processors, table,
                                   grad_out, g_stride_b, g_stride_r, grad_in, gi_stride_b, gi_stride_r, stream);
}
