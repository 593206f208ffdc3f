// Logits, and token logprobs, from hidden states and an output weight in 8-bit integers, one fp32 scale
// per row of either:
//   x[r, v]   = (float(sum_k h8[r, k] w8[v, k]) * ws[v]) * hs[r]
//   logprob_t = (x_t - m) - log(sum_v exp(x_v - m)),  0 for targets outside [vs, ve)
// on the tile loop of the other hidden-state paths (lce_tile.h), whose stages hold the same 128 bytes
// of a row and whose accumulators are 32-bit integers: the sum is exact and its rounding to fp32 (above
// 2^24) is the first one.  The target's logit is therefore the tile's own.
//
// Bound by the matrix cores and what feeds them, few rows by the weight's bytes.  [16376, 4096] x [151936, 4096]:
// logprobs 7.66 to 8.1 ms from card to card, 2.5 to 2.66 POP/s (a library product alone 2.13 POP/s).  Logits
// of [2048, 4096] x [151936, 4096] in bf16, 622 MB of them: 1.05 to 1.10 ms, 2.3 to 2.4 POP/s; in fp32 1.17, with an odd
// vocabulary, whose rows no 16 bytes divide, 1.54 (words stored one by one).  Of 64 rows: logits 131 us,
// logprobs 124 us, 4.9 and 5.0 TB/s.

#include "lce_tile.h"

#pragma clang fp contract(off)

using namespace mirl;

namespace {

// |products| <= 2^14, so sums of fewer than 2^17 of them stay inside 32 bits (in whole steps of 256).
constexpr int64_t kMaxHidden = (int64_t(1) << 17) - 256;

int operands(LceParams& P, const int8_t* hidden8, const float* hidden_scale, int64_t T, int64_t Hd, int64_t ldh,
             const int8_t* weight8, const float* weight_scale, int64_t V, int64_t ldw) {
  MIRL_REQUIRE(T >= 0 && V > 0 && Hd > 0, "invalid shape T=%lld V=%lld H=%lld", (long long)T, (long long)V, (long long)Hd);
  MIRL_REQUIRE(Hd <= kMaxHidden, "hidden size %lld: sums of more than %lld products may pass 32 bits", (long long)Hd,
               (long long)kMaxHidden);
  // buffer ranges of one 256-row tile are 32-bit byte counts
  MIRL_REQUIRE(ldh < (int64_t(1) << 22) && ldw < (int64_t(1) << 22),
               "row strides (%lld, %lld) must be below 2^22 elements", (long long)ldh, (long long)ldw);
  MIRL_REQUIRE(V < (int64_t(1) << 31) && T < (int64_t(1) << 31), "sizes exceed 2^31-1");
  const int64_t padded = padded_hidden(Hd, 1);
  // A weight without gaps may have rows of any whole words: what a row's last piece holds of the next row
  // meets the hidden states' zeros, and the last row's is cut off word by word by the buffer's range.
  const bool packed = Hd % 4 == 0 && ldw == Hd && (reinterpret_cast<uintptr_t>(weight8) & 3u) == 0;
  const bool pieces = Hd % 16 == 0 && ldw % 16 == 0 && ldw >= Hd && (reinterpret_cast<uintptr_t>(weight8) & 15u) == 0;
  MIRL_REQUIRE(ldh % 16 == 0 && ldh >= padded && (packed || pieces),
               "hidden size %lld and row strides (%lld, %lld) must be multiples of 16 and the weight 16-byte aligned (or its "
               "rows whole words without gaps), the hidden states' rows padded to %lld",
               (long long)Hd, (long long)ldh, (long long)ldw, (long long)padded);
  if (T == 0) return MIRL_OK;
  MIRL_REQUIRE(hidden8 && hidden_scale && weight8 && weight_scale, "null pointer argument");
  MIRL_REQUIRE((reinterpret_cast<uintptr_t>(hidden8) & 15u) == 0, "hidden states must be 16-byte aligned");
  P.h = hidden8;
  P.w = weight8;
  P.ldh = ldh;
  P.ldw = ldw;
  P.V = V;
  P.Hd = padded;
  P.Hw = Hd;
  P.nrows = T;
  P.bsz = 1;
  P.row_scale = hidden_scale;
  P.col_scale = weight_scale;
  return MIRL_OK;
}

}  // namespace

extern "C" int mirl_linear_ce_int8_fwd(const int8_t* hidden8, const float* hidden_scale, int64_t T, int64_t Hd, int64_t ldh,
                                       const int8_t* weight8, const float* weight_scale, int64_t V, int64_t ldw,
                                       int64_t bsz, const int64_t* target, int64_t t_stride_b, int64_t t_stride_s,
                                       int64_t vocab_start, int64_t vocab_end, float* out, int64_t o_stride_b,
                                       int64_t o_stride_s, float* workspace, void* stream) {
  clear_error();
  LceParams P{};
  MIRL_REQUIRE(bsz > 0, "invalid batch size %lld", (long long)bsz);
  MIRL_REQUIRE(T % bsz == 0, "row count %lld is not a multiple of the batch size %lld", (long long)T, (long long)bsz);
  // (a wave merges a row's parts, and a launch holds fewer than 2^32 threads)
  MIRL_REQUIRE(T < (int64_t(1) << 26), "%lld rows: fewer than 2^26 are scored in a call", (long long)T);
  if (int e = operands(P, hidden8, hidden_scale, T, Hd, ldh, weight8, weight_scale, V, ldw)) return e;
  if (T == 0) return MIRL_OK;
  MIRL_REQUIRE(target && out && workspace, "null pointer argument");
  P.bsz = bsz;
  P.target = target;
  P.tsb = t_stride_b;
  P.tss = t_stride_s;
  P.vs = vocab_start;
  P.ve = vocab_end;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t tiles = launch_fwd_x<I8>(P, workspace, st);
  MIRL_REQUIRE(tiles < (int64_t(1) << 24), "too many tiles");
  auto merge = [&](auto w) {
    constexpr int W = decltype(w)::value;
    hipLaunchKernelGGL(lce_merge_kernel<W>, dim3((unsigned)(W == 1 ? ceil_div(T, 4) : T)), dim3(256), 0, st, P.part, P.xt,
                       int64_t(0), T, P.n_nt, bsz, target, t_stride_b, t_stride_s, vocab_start, vocab_end, V, out, o_stride_b,
                       o_stride_s, static_cast<float*>(nullptr), static_cast<const int64_t*>(nullptr));
  };
  if (T <= kJoinRows)
    merge(std::integral_constant<int, 4>{});
  else
    merge(std::integral_constant<int, 1>{});
  return check_launch("mirl_linear_ce_int8_fwd");
}

extern "C" int mirl_int8_logits(const int8_t* hidden8, const float* hidden_scale, int64_t T, int64_t Hd, int64_t ldh,
                                const int8_t* weight8, const float* weight_scale, int64_t V, int64_t ldw, void* out,
                                int out_dtype, int64_t ldo, void* stream) {
  clear_error();
  LceParams P{};
  MIRL_REQUIRE(out_dtype == MIRL_DTYPE_F32 || out_dtype == MIRL_DTYPE_BF16 || out_dtype == MIRL_DTYPE_F16,
               "unsupported logits dtype code %d", out_dtype);
  if (int e = operands(P, hidden8, hidden_scale, T, Hd, ldh, weight8, weight_scale, V, ldw)) return e;
  if (T == 0) return MIRL_OK;
  MIRL_REQUIRE(out != nullptr, "null pointer argument");
  MIRL_REQUIRE(T == 1 || ldo >= V, "row stride %lld of the logits is below V=%lld", (long long)ldo, (long long)V);
  if (out_dtype == MIRL_DTYPE_F32) {
    P.C = static_cast<float*>(out);
    P.ldc = ldo;
  } else {
    P.Cb = static_cast<uint16_t*>(out);
    P.cb_f16 = out_dtype == MIRL_DTYPE_F16;
    P.ldcb = ldo;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t tiles = out_dtype == MIRL_DTYPE_F32    ? launch_fwd_x<I8, kLogits, F32>(P, nullptr, st)
                        : out_dtype == MIRL_DTYPE_BF16 ? launch_fwd_x<I8, kLogits, BF16>(P, nullptr, st)
                                                       : launch_fwd_x<I8, kLogits, F16>(P, nullptr, st);
  MIRL_REQUIRE(tiles < (int64_t(1) << 24), "too many tiles");
  return check_launch("mirl_int8_logits");
}
