// Token logprobs straight from hidden states and the output (LM-head) weight:
// the logits tile H[rows] . W[cols]^T is formed on the MFMA units and reduced
// in the same kernel, so the [T, V] logits are never written.
//
// Semantics follow nemo_rl/distributed/model_utils.py:2541-2745
// (from_parallel_hidden_states_to_logprobs, ChunkedDistributedHiddenStatesToLogprobs)
// with a vocab group of size 1:
//   logits    = bf16(H . W^T)                (the reference's bf16 matmul output)
//   logprob_t = (x_t - m) - log(sum_v exp(x_v - m)),  0 for targets outside [vs, ve)
//   backward  G = (onehot(t) - softmax(x)) * g,  dH = G . W,  dW = G^T . H
// The forward kernel writes, per row and per 256-column tile, the tile's
// (max, sum exp(x - max)) and the target logit; a merge kernel combines the
// tiles of a row.  The gradient kernel recomputes a logits tile and writes the
// bf16 G tile and its transpose; the two products that consume G run on the
// same tile loop as a plain GEMM.  Row counts may live on the device (the
// backward's active rows): the kernels read them and skip what lies past them,
// so the host never waits for them.
//
// Tile: 256 rows x 256 columns per 256-thread workgroup.  Each wave owns a
// 128 x 128 quarter as 8 x 8 v_mfma_f32_16x16x32 tiles (256 fp32 accumulators
// per lane).  The hidden dimension streams through two LDS stages
// of 64 elements (64 KB each: 256 rows of H and 256 rows of W, 128 B per row),
// filled by direct global->LDS loads (buffer_load_dwordx4 ... lds) one stage
// ahead of the MFMAs: no staging registers and no LDS store instructions sit
// between the loads and the MFMAs, and the only waits are one vmcnt + barrier
// per stage.  Each row of a stage is one 128-byte line of H or W.  A row's
// eight 16-byte chunks are XOR-swizzled by (row / 2) % 8 (see lds_off), so the
// 16 rows read by one pass of an MFMA operand load fall in distinct banks.
//
// The MFMA lane layouts (checked on gfx950) stand at Mma<E>.

#include "lce_tile.h"

#pragma clang fp contract(off)

namespace mirl {
namespace {

// dst[c][r] = bf16(src[r][c]) for r < R, c < C, and dst[c][r] = 0 for
// R <= r < Rp (src of dtype ES, bf16 or fp16; dst rows of stride ldd >= Rp),
// R = min(R, *count) when count is given.  64 x 64 tiles through LDS, moved
// as 16-byte pieces (eight elements of a row in, eight of a column out) where
// the pointers, strides and tile edges allow, element by element elsewhere.
template <class ES>
__global__ __launch_bounds__(256) void transpose_bf16_kernel(const uint16_t* __restrict__ src,
                                                             int64_t R, int64_t C, int64_t lds,
                                                             uint16_t* __restrict__ dst,
                                                             int64_t ldd, int64_t Rp,
                                                             int64_t n_ct,
                                                             const int64_t* __restrict__ count) {
  // row pitch 66 elements (33 words): the eight rows 8 apart that a wave's
  // column reads touch start in different LDS banks
  constexpr int kP = 66;
  __shared__ uint16_t tile[64 * kP];
  if (count != nullptr && *count < R) R = *count;
  const int64_t tr = blockIdx.x / n_ct, tc = blockIdx.x - tr * n_ct;
  const int64_t r0 = tr * 64, c0 = tc * 64;
  const bool vin = ((lds & 7) | (reinterpret_cast<uintptr_t>(src) & 15)) == 0;
  const bool vout = ((ldd & 7) | (reinterpret_cast<uintptr_t>(dst) & 15)) == 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int idx = (int)threadIdx.x + 256 * k, lr = idx >> 3, cg = (idx & 7) * 8;
    const int64_t r = r0 + lr, c = c0 + cg;
    uint32_t w[4];
    if (vin && r < R && c + 8 <= C) {
      const vu4 q = *reinterpret_cast<const vu4*>(src + r * lds + c);
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = (r < R && c + 2 * j < C) ? src[r * lds + c + 2 * j] : 0u;
        const uint32_t hi = (r < R && c + 2 * j + 1 < C) ? src[r * lds + c + 2 * j + 1] : 0u;
        w[j] = lo | (hi << 16);
      }
    }
    if constexpr (std::is_same<ES, F16>::value) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = (uint32_t)bits_of<BF16>(value_of<F16>((uint16_t)(w[j] & 0xffffu))) |
               ((uint32_t)bits_of<BF16>(value_of<F16>((uint16_t)(w[j] >> 16))) << 16);
    }
    // (lr * 66 + cg) elements = a whole number of 4-byte words
    uint32_t* t32 = reinterpret_cast<uint32_t*>(tile + lr * kP + cg);
#pragma unroll
    for (int j = 0; j < 4; ++j) t32[j] = w[j];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int idx = (int)threadIdx.x + 256 * k, lc = idx >> 3, rg = (idx & 7) * 8;
    const int64_t c = c0 + lc, r = r0 + rg;
    if (c >= C) continue;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = (uint32_t)tile[(rg + 2 * j) * kP + lc] | ((uint32_t)tile[(rg + 2 * j + 1) * kP + lc] << 16);
    uint16_t* d = dst + c * ldd + r;
    if (vout && r + 8 <= Rp) {
      *reinterpret_cast<vu4*>(d) = vu4{w[0], w[1], w[2], w[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r + i < Rp) d[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// dst[c][r] = src[r][c] for r < R, c < C, and dst[c][r] = 0 for R <= r < Rp
// (fp32; dst rows of stride ldd >= Rp), R = min(R, *count - count_off) when
// count is given.  64 x 64 tiles through LDS, moved as 16-byte pieces (four
// elements of a row in, four of a column out) where the pointers, strides and
// tile edges allow, element by element elsewhere.
__global__ __launch_bounds__(256) void transpose_f32_kernel(const float* __restrict__ src, int64_t R,
                                                            int64_t C, int64_t lds,
                                                            float* __restrict__ dst, int64_t ldd,
                                                            int64_t Rp, int64_t n_ct,
                                                            const int64_t* __restrict__ count,
                                                            int64_t count_off) {
  // row pitch 65 words: a wave's row pieces and column reads each fall in
  // distinct LDS banks
  constexpr int kP = 65;
  __shared__ float tile[64 * kP];
  if (count != nullptr) {
    const int64_t c = *count - count_off;
    if (c < R) R = c < 0 ? 0 : c;
  }
  const int64_t tr = blockIdx.x / n_ct, tc = blockIdx.x - tr * n_ct;
  const int64_t r0 = tr * 64, c0 = tc * 64;
  const bool vin = ((lds & 3) | (reinterpret_cast<uintptr_t>(src) & 15)) == 0;
  const bool vout = ((ldd & 3) | (reinterpret_cast<uintptr_t>(dst) & 15)) == 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int idx = (int)threadIdx.x + 256 * k, lr = idx >> 4, cg = (idx & 15) * 4;
    const int64_t r = r0 + lr, c = c0 + cg;
    float w[4];
    if (vin && r < R && c + 4 <= C) {
      const float4 q = *reinterpret_cast<const float4*>(src + r * lds + c);
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (r < R && c + j < C) ? src[r * lds + c + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[lr * kP + cg + j] = w[j];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int idx = (int)threadIdx.x + 256 * k, lc = idx >> 4, rg = (idx & 15) * 4;
    const int64_t c = c0 + lc, r = r0 + rg;
    if (c >= C) continue;
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = tile[(rg + i) * kP + lc];
    float* d = dst + c * ldd + r;
    if (vout && r + 4 <= Rp) {
      *reinterpret_cast<float4*>(d) = make_float4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + i < Rp) d[i] = w[i];
    }
  }
}

// out[r(m)][n] = EO(sum over s of part[s][m][n]) (EO bf16, fp16 or fp32), summed in split order,
// with r(m) = out_rows[m] when a row map is given (rows mapped outside
// [0, out_nrows) are skipped) and m otherwise; with a count, rows
// m >= *count - count_off are written as zeros without reading.  VEC
// consecutive elements per thread (N and ld multiples of VEC).
template <int VEC, class EO>
__global__ __launch_bounds__(256) void sum_splits_kernel(const float* __restrict__ part,
                                                         int64_t n_ks, int64_t M, int64_t N,
                                                         int64_t ld, void* __restrict__ out,
                                                         int64_t ldo,
                                                         const int64_t* __restrict__ out_rows,
                                                         int64_t out_nrows,
                                                         const int64_t* __restrict__ count,
                                                         int64_t count_off) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
  if (i >= M * N) return;
  const int64_t m = i / N, n = i - m * N;
  int64_t r = m;
  if (out_rows != nullptr) {
    r = out_rows[m];
    if (r < 0 || r >= out_nrows) return;
  }
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  if (count == nullptr || m < *count - count_off) {
    for (int64_t s = 0; s < n_ks; ++s) {
      const float* src = part + (s * M + m) * ld + n;
      if constexpr (VEC == 4) {
        const float4 q = *reinterpret_cast<const float4*>(src);
        acc[0] += q.x;
        acc[1] += q.y;
        acc[2] += q.z;
        acc[3] += q.w;
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += src[e];
      }
    }
  }
  if constexpr (std::is_same<EO, F32>::value) {
    float* dst = static_cast<float*>(out) + r * ldo + n;
    if constexpr (VEC == 4) {
      *reinterpret_cast<float4*>(dst) = float4{acc[0], acc[1], acc[2], acc[3]};
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) dst[e] = acc[e];
    }
  } else {
    uint16_t* dst = static_cast<uint16_t*>(out) + r * ldo + n;
    if constexpr (VEC == 4) {
      const uint32_t lo = (uint32_t)bits_of<EO>(acc[0]) | ((uint32_t)bits_of<EO>(acc[1]) << 16);
      const uint32_t hi = (uint32_t)bits_of<EO>(acc[2]) | ((uint32_t)bits_of<EO>(acc[3]) << 16);
      *reinterpret_cast<uint2*>(dst) = uint2{lo, hi};
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) dst[e] = bits_of<EO>(acc[e]);
    }
  }
}

// The rows r = (s, b) = (r / bsz, r % bsz) whose upstream gradient is not zero, in
// order, then the others from the end backwards: perm, the rows' gradients and the
// count of the first kind.  One workgroup, 8 x 1024 rows a step (their loads in
// flight together, a ballot and a sum over 16 waves per 1024).  With the gather below
// it takes the place of a stable sort, a sum and six gathers of the library: step of
// 137 rows x [1355, 4096] fp16 356 -> 248 us (host-bound), of 115 rows x [11749, 4096]
// bf16 441 -> 337; nothing to see at 16384 rows.
constexpr int kActThreads = 1024;
__global__ __launch_bounds__(kActThreads) void lce_active_rows_kernel(
    const float* __restrict__ g, int64_t gsb, int64_t gss, uint32_t T, uint32_t bsz,
    int64_t* __restrict__ perm, float* __restrict__ g_a, int64_t* __restrict__ count) {
  constexpr int NW = kActThreads / kWave, U = 8;
  __shared__ uint32_t wsum[2][NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t base = 0;  // active rows before this step
  for (uint32_t r0 = 0; r0 < T; r0 += U * kActThreads) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * kActThreads + tid;
      const uint32_t s = r / bsz, b = r - s * bsz;
      v[u] = r < T ? g[(int64_t)b * gsb + (int64_t)s * gss] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * kActThreads + tid;
      const bool act = r < T && v[u] != 0.f;
      const uint64_t bal = __ballot(act);
      // the two buffers alternate, so one barrier a round separates a round's
      // writes from the reads of the round before last
      if (lane == 0) wsum[u & 1][wave] = (uint32_t)__popcll(bal);
      __syncthreads();
      uint32_t before = base + (uint32_t)__popcll(bal & ((1ull << lane) - 1ull));
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const uint32_t n = wsum[u & 1][w];
        before += w < wave ? n : 0u;
        base += n;
      }
      if (r < T) {
        const uint32_t at = act ? before : T - 1 - (r - before);
        perm[at] = r;
        g_a[at] = v[u];
      }
    }
  }
  if (tid == 0) *count = base;
}

// Row m of the permuted targets and statistics and, for m < *count, of the permuted
// hidden states (row_units units of UNIT per row; rows past the count stay as they
// are: every kernel stops at the count).  One workgroup per row, up to kGatherGrid of
// them: a launch holds fewer than 2^32 threads.
constexpr int64_t kGatherGrid = int64_t(1) << 20;
template <class UNIT>
__global__ __launch_bounds__(256) void lce_gather_rows_kernel(
    const int64_t* __restrict__ perm, const int64_t* __restrict__ count, int64_t T, uint32_t bsz,
    const int64_t* __restrict__ target, int64_t tsb, int64_t tss, const float* __restrict__ stats,
    const UNIT* __restrict__ hidden, int64_t row_units, int64_t ld_units, int64_t* __restrict__ tgt_a,
    float* __restrict__ st_a, UNIT* __restrict__ h_a) {
  for (int64_t m = blockIdx.x; m < T; m += kGatherGrid) {
    const uint32_t r = (uint32_t)perm[m];
    const bool live = m < *count;
    if (threadIdx.x == 0) {
      const uint32_t s = r / bsz, b = r - s * bsz;
      tgt_a[m] = target[(int64_t)b * tsb + (int64_t)s * tss];
      st_a[2 * m] = stats[2 * (int64_t)r];
      st_a[2 * m + 1] = stats[2 * (int64_t)r + 1];
    }
    if (!live) continue;
    const UNIT* src = hidden + (int64_t)r * ld_units;
    UNIT* dst = h_a + m * row_units;
    for (int64_t k = threadIdx.x; k < row_units; k += 256) dst[k] = src[k];
  }
}

int check_common(const void* hidden, int64_t T, int64_t Hd, int64_t ldh, const void* weight,
                 int64_t V, int64_t ldw, const int64_t* target, int64_t bsz) {
  MIRL_REQUIRE(hidden && weight && target, "null pointer argument");
  MIRL_REQUIRE(T >= 0 && V > 0 && Hd > 0 && bsz > 0, "invalid shape T=%lld V=%lld H=%lld B=%lld",
               (long long)T, (long long)V, (long long)Hd, (long long)bsz);
  MIRL_REQUIRE(T % bsz == 0, "row count %lld is not a multiple of the batch size %lld",
               (long long)T, (long long)bsz);
  MIRL_REQUIRE(Hd % (kStages * kSK) == 0, "hidden size %lld must be a multiple of %d", (long long)Hd,
               kStages * kSK);
  MIRL_REQUIRE(ldh < (int64_t(1) << 22) && ldw < (int64_t(1) << 22),
               "row strides (%lld, %lld) must be below 2^22 elements", (long long)ldh, (long long)ldw);
  MIRL_REQUIRE(ldh % 8 == 0 && ldw % 8 == 0 && ldh >= Hd && ldw >= Hd,
               "row strides (%lld, %lld) must be multiples of 8 elements and >= the hidden size",
               (long long)ldh, (long long)ldw);
  MIRL_REQUIRE((reinterpret_cast<uintptr_t>(hidden) & 15u) == 0 &&
                   (reinterpret_cast<uintptr_t>(weight) & 15u) == 0,
               "hidden states and weight must be 16-byte aligned");
  MIRL_REQUIRE(V < (int64_t(1) << 31) && T < (int64_t(1) << 31), "sizes exceed 2^31-1");
  return MIRL_OK;
}

}  // namespace
}  // namespace mirl

using namespace mirl;

extern "C" int64_t mirl_linear_ce_workspace_elems(int64_t T, int64_t V) {
  if (T <= 0 || V <= 0) return 0;
  return T * ceil_div(V, kBN) * 2 + T;
}

static bool lce_dtype_ok(int dtype) { return dtype == MIRL_DTYPE_BF16 || dtype == MIRL_DTYPE_F16; }

extern "C" int mirl_linear_ce_fwd(const void* hidden, int dtype, int64_t T, int64_t Hd, int64_t ldh,
                                  const void* weight, int64_t V, int64_t ldw, int64_t bsz,
                                  const int64_t* target, int64_t t_stride_b, int64_t t_stride_s,
                                  int64_t vocab_start, int64_t vocab_end, float* out,
                                  int64_t o_stride_b, int64_t o_stride_s, float* row_stats,
                                  float* workspace, void* stream) {
  clear_error();
  MIRL_REQUIRE(lce_dtype_ok(dtype), "hidden states and weight must be bf16 or fp16 (dtype code %d)",
               dtype);
  if (int e = check_common(hidden, T, Hd, ldh, weight, V, ldw, target, bsz)) return e;
  if (T == 0) return MIRL_OK;
  MIRL_REQUIRE(out && workspace, "null pointer argument");
  hipStream_t st = static_cast<hipStream_t>(stream);
  LceParams P{};
  P.h = static_cast<const uint16_t*>(hidden);
  P.w = static_cast<const uint16_t*>(weight);
  P.ldh = ldh;
  P.ldw = ldw;
  P.V = V;
  P.Hd = Hd;
  P.row0 = 0;
  P.nrows = T;
  P.bsz = bsz;
  P.target = target;
  P.tsb = t_stride_b;
  P.tss = t_stride_s;
  P.vs = vocab_start;
  P.ve = vocab_end;
  P.n_mt = ceil_div(T, kBM);
  P.n_nt = ceil_div(V, kBN);
  P.part = workspace;
  P.xt = workspace + T * P.n_nt * 2;
  const int64_t grid = ceil_div(P.n_mt * P.n_nt, kXcds) * kXcds;
  MIRL_REQUIRE(grid < (int64_t(1) << 31), "too many tiles");
  if (dtype == MIRL_DTYPE_BF16)
    hipLaunchKernelGGL((lce_tile_kernel<kFwd, BF16>), dim3((unsigned)grid), dim3(kThreads), 0, st, P);
  else
    hipLaunchKernelGGL((lce_tile_kernel<kFwd, F16>), dim3((unsigned)grid), dim3(kThreads), 0, st, P);
  hipLaunchKernelGGL(lce_merge_kernel<1>, dim3((unsigned)ceil_div(T, 4)), dim3(256), 0, st, P.part,
                     P.xt, (int64_t)0, T, P.n_nt, bsz, target, t_stride_b, t_stride_s,
                     vocab_start, vocab_end, V, out, o_stride_b, o_stride_s, row_stats, nullptr);
  return check_launch("mirl_linear_ce_fwd");
}

extern "C" int mirl_linear_ce_grad(const void* hidden, int dtype, int64_t T, int64_t Hd, int64_t ldh,
                                   const void* weight, int64_t V, int64_t ldw, int64_t bsz,
                                   const int64_t* target, int64_t t_stride_b,
                                   int64_t t_stride_s, int64_t vocab_start, int64_t vocab_end,
                                   const float* row_stats, const float* grad_out,
                                   int64_t g_stride_b, int64_t g_stride_s, int64_t row0,
                                   int64_t nrows, void* grad_logits, int64_t ldg,
                                   void* grad_logits_t, int64_t ldgt, const int64_t* row_count,
                                   void* stream) {
  clear_error();
  MIRL_REQUIRE(lce_dtype_ok(dtype), "hidden states and weight must be bf16 or fp16 (dtype code %d)",
               dtype);
  if (int e = check_common(hidden, T, Hd, ldh, weight, V, ldw, target, bsz)) return e;
  MIRL_REQUIRE(row0 >= 0 && nrows >= 0 && row0 + nrows <= T, "row range [%lld, %lld) outside [0, %lld)",
               (long long)row0, (long long)(row0 + nrows), (long long)T);
  if (nrows == 0) return MIRL_OK;
  MIRL_REQUIRE(row_stats && grad_out && grad_logits, "null pointer argument");
  MIRL_REQUIRE(ldg >= V, "gradient row stride %lld is smaller than V=%lld", (long long)ldg,
               (long long)V);
  // the transposed tiles cover whole 256-row tiles, written as 16-byte vectors
  MIRL_REQUIRE(grad_logits_t == nullptr ||
                   (ldgt >= ceil_div(nrows, kBM) * kBM && ldgt % 8 == 0 &&
                    (reinterpret_cast<uintptr_t>(grad_logits_t) & 15u) == 0),
               "transposed gradient: row stride %lld must cover %lld rows in whole 256-row tiles, "
               "be a multiple of 8 elements and start 16-byte aligned",
               (long long)ldgt, (long long)nrows);
  hipStream_t st = static_cast<hipStream_t>(stream);
  LceParams P{};
  P.h = static_cast<const uint16_t*>(hidden);
  P.w = static_cast<const uint16_t*>(weight);
  P.ldh = ldh;
  P.ldw = ldw;
  P.V = V;
  P.Hd = Hd;
  P.row0 = row0;
  P.nrows = nrows;
  P.bsz = bsz;
  P.target = target;
  P.tsb = t_stride_b;
  P.tss = t_stride_s;
  P.vs = vocab_start;
  P.ve = vocab_end;
  P.n_mt = ceil_div(nrows, kBM);
  P.n_nt = ceil_div(V, kBN);
  P.stats = row_stats;
  P.g = grad_out;
  P.gsb = g_stride_b;
  P.gss = g_stride_s;
  P.G = static_cast<uint16_t*>(grad_logits);
  P.ldg = ldg;
  P.Gt = static_cast<uint16_t*>(grad_logits_t);
  P.ldgt = ldgt;
  P.count = row_count;
  const int64_t grid = ceil_div(P.n_mt * P.n_nt, kXcds) * kXcds;
  MIRL_REQUIRE(grid < (int64_t(1) << 31), "too many tiles");
  if (dtype == MIRL_DTYPE_BF16)
    hipLaunchKernelGGL((lce_tile_kernel<kGrad, BF16>), dim3((unsigned)grid), dim3(kThreads), 0, st, P);
  else
    hipLaunchKernelGGL((lce_tile_kernel<kGrad, F16>), dim3((unsigned)grid), dim3(kThreads), 0, st, P);
  return check_launch("mirl_linear_ce_grad");
}

extern "C" int mirl_gemm_bf16_abt(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M,
                                  int64_t N, int64_t K, int64_t k_splits, float* C, int64_t ldc,
                                  int accumulate, void* Cb, int64_t ldcb, int cb_dtype,
                                  const int64_t* count, int64_t count_off, int count_axis,
                                  int64_t final_at, void* stream) {
  clear_error();
  MIRL_REQUIRE(Cb == nullptr || lce_dtype_ok(cb_dtype), "the 16-bit output must be bf16 or fp16 (dtype code %d)",
               cb_dtype);
  MIRL_REQUIRE(M >= 0 && N >= 0 && K > 0 && k_splits >= 1, "invalid shape M=%lld N=%lld K=%lld splits=%lld",
               (long long)M, (long long)N, (long long)K, (long long)k_splits);
  if (M == 0 || N == 0) return MIRL_OK;
  MIRL_REQUIRE(A && B && (C || Cb), "null pointer argument");
  const int64_t kstep = (int64_t)kStages * kSK;
  MIRL_REQUIRE(K % kstep == 0, "reduction length %lld must be a multiple of %lld", (long long)K,
               (long long)kstep);
  const int64_t kb = ceil_div(ceil_div(K, k_splits), kstep) * kstep;
  const int64_t n_ks = ceil_div(K, kb);
  MIRL_REQUIRE(n_ks == k_splits,
               "%lld splits of K=%lld in ranges of %lld leave %lld non-empty (choose a split count "
               "that divides into whole 128-element ranges)",
               (long long)k_splits, (long long)K, (long long)kb, (long long)n_ks);
  MIRL_REQUIRE(count_axis == MIRL_COUNT_ROWS || count_axis == MIRL_COUNT_K, "invalid count axis %d",
               count_axis);
  const bool both = C != nullptr && Cb != nullptr;
  MIRL_REQUIRE(!both || (count != nullptr && count_axis == MIRL_COUNT_K && n_ks == 1),
               "an fp32 and a bf16 output together take a reduction-length count and one split");
  MIRL_REQUIRE(Cb == nullptr || (n_ks == 1 && (!accumulate || both)),
               "a bf16 output takes one split and accumulates only over the fp32 output");
  MIRL_REQUIRE(!accumulate || n_ks == 1, "accumulation takes one split");
  MIRL_REQUIRE(lda % 8 == 0 && ldb % 8 == 0 && lda >= K && ldb >= K,
               "row strides (%lld, %lld) must be multiples of 8 elements and >= K", (long long)lda,
               (long long)ldb);
  MIRL_REQUIRE((reinterpret_cast<uintptr_t>(A) & 15u) == 0 && (reinterpret_cast<uintptr_t>(B) & 15u) == 0,
               "operands must be 16-byte aligned");
  // buffer ranges of one 256-row tile are 32-bit byte counts
  MIRL_REQUIRE(kBM * lda * 2 < (int64_t(1) << 31) && kBN * ldb * 2 < (int64_t(1) << 31),
               "row strides (%lld, %lld) too large", (long long)lda, (long long)ldb);
  MIRL_REQUIRE(M < (int64_t(1) << 31) && N < (int64_t(1) << 31), "sizes exceed 2^31-1");
  MIRL_REQUIRE(C == nullptr || ldc >= N, "output row stride %lld is smaller than N=%lld",
               (long long)ldc, (long long)N);
  MIRL_REQUIRE(Cb == nullptr || ldcb >= N, "output row stride %lld is smaller than N=%lld",
               (long long)ldcb, (long long)N);
  LceParams P{};
  P.h = static_cast<const uint16_t*>(A);
  P.w = static_cast<const uint16_t*>(B);
  P.ldh = lda;
  P.ldw = ldb;
  P.V = N;
  P.Hd = K;
  P.row0 = 0;
  P.nrows = M;
  P.n_mt = ceil_div(M, kBM);
  P.n_nt = ceil_div(N, kBN);
  P.n_ks = n_ks;
  P.kb_len = kb;
  P.C = C;
  P.Cb = static_cast<uint16_t*>(Cb);
  P.cb_f16 = cb_dtype == MIRL_DTYPE_F16;
  P.ldc = ldc;
  P.ldcb = ldcb;
  P.accumulate = accumulate;
  P.count = count;
  P.count_off = count_off;
  P.count_axis = count_axis;
  P.final_at = final_at;
  const int64_t grid = ceil_div(P.n_mt * P.n_nt * n_ks, kXcds) * kXcds;
  MIRL_REQUIRE(grid < (int64_t(1) << 31), "too many tiles");
  hipLaunchKernelGGL((lce_tile_kernel<kGemm, BF16>), dim3((unsigned)grid), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), P);
  return check_launch("mirl_gemm_bf16_abt");
}

extern "C" int mirl_sum_splits_bf16(const float* part, int64_t k_splits, int64_t M, int64_t N,
                                    int64_t ld, void* out, int64_t ldo, int out_dtype,
                                    const int64_t* out_rows, int64_t out_nrows,
                                    const int64_t* count, int64_t count_off, void* stream) {
  clear_error();
  MIRL_REQUIRE(lce_dtype_ok(out_dtype) || out_dtype == MIRL_DTYPE_F32,
               "the output must be bf16, fp16 or fp32 (dtype code %d)", out_dtype);
  MIRL_REQUIRE(M >= 0 && N >= 0 && k_splits >= 1 && ld >= N && ldo >= N, "invalid shape");
  if (M == 0 || N == 0) return MIRL_OK;
  MIRL_REQUIRE(part && out, "null pointer argument");
  MIRL_REQUIRE(out_rows == nullptr || out_nrows >= 0, "invalid output row count");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uintptr_t out_align = out_dtype == MIRL_DTYPE_F32 ? 15u : 7u;  // 4 elements
  const bool vec4 = N % 4 == 0 && ld % 4 == 0 && ldo % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(part) & 15u) == 0 &&
                    (reinterpret_cast<uintptr_t>(out) & out_align) == 0;
  auto launch = [&](auto vec_c, auto eo) {
    constexpr int VEC = decltype(vec_c)::value;
    using EO = decltype(eo);
    hipLaunchKernelGGL((sum_splits_kernel<VEC, EO>), dim3((unsigned)ceil_div(M * N / VEC, 256)),
                       dim3(256), 0, st, part, k_splits, M, N, ld, out, ldo, out_rows, out_nrows,
                       count, count_off);
  };
  using V4 = std::integral_constant<int, 4>;
  using V1 = std::integral_constant<int, 1>;
  if (out_dtype == MIRL_DTYPE_BF16) {
    if (vec4) launch(V4{}, BF16{}); else launch(V1{}, BF16{});
  } else if (out_dtype == MIRL_DTYPE_F16) {
    if (vec4) launch(V4{}, F16{}); else launch(V1{}, F16{});
  } else {
    if (vec4) launch(V4{}, F32{}); else launch(V1{}, F32{});
  }
  return check_launch("mirl_sum_splits_bf16");
}

extern "C" int mirl_transpose_bf16(const void* src, int src_dtype, int64_t R, int64_t C,
                                   int64_t lds, void* dst, int64_t ldd, int64_t R_pad,
                                   const int64_t* count, void* stream) {
  clear_error();
  MIRL_REQUIRE(lce_dtype_ok(src_dtype), "the source must be bf16 or fp16 (dtype code %d)", src_dtype);
  MIRL_REQUIRE(R >= 0 && C >= 0 && R_pad >= R && lds >= C && ldd >= R_pad, "invalid shape");
  if (C == 0 || R_pad == 0) return MIRL_OK;
  MIRL_REQUIRE(src && dst, "null pointer argument");
  const int64_t n_rt = ceil_div(R_pad, 64), n_ct = ceil_div(C, 64);
  MIRL_REQUIRE(n_rt * n_ct < (int64_t(1) << 31), "too many tiles");
  auto launch = [&](auto es) {
    using ES = decltype(es);
    hipLaunchKernelGGL((transpose_bf16_kernel<ES>), dim3((unsigned)(n_rt * n_ct)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), static_cast<const uint16_t*>(src), R, C,
                       lds, static_cast<uint16_t*>(dst), ldd, R_pad, n_ct, count);
  };
  if (src_dtype == MIRL_DTYPE_BF16) launch(BF16{}); else launch(F16{});
  return check_launch("mirl_transpose_bf16");
}

extern "C" int mirl_gemm_f32_abt(const float* A, int64_t lda, const float* B, int64_t ldb, int64_t M,
                                 int64_t N, int64_t K, int64_t k_splits, float* C, int64_t ldc,
                                 int accumulate, const int64_t* count, int64_t count_off,
                                 int count_axis, void* stream) {
  clear_error();
  MIRL_REQUIRE(M >= 0 && N >= 0 && K > 0 && k_splits >= 1, "invalid shape M=%lld N=%lld K=%lld splits=%lld",
               (long long)M, (long long)N, (long long)K, (long long)k_splits);
  if (M == 0 || N == 0) return MIRL_OK;
  MIRL_REQUIRE(A && B && C, "null pointer argument");
  const int64_t kstep = (int64_t)kStages * (kRowBytes / 4);
  MIRL_REQUIRE(K % kstep == 0, "reduction length %lld must be a multiple of %lld", (long long)K,
               (long long)kstep);
  const int64_t kb = ceil_div(ceil_div(K, k_splits), kstep) * kstep;
  const int64_t n_ks = ceil_div(K, kb);
  MIRL_REQUIRE(n_ks == k_splits,
               "%lld splits of K=%lld in ranges of %lld leave %lld non-empty (choose a split count "
               "that divides into whole 64-element ranges)",
               (long long)k_splits, (long long)K, (long long)kb, (long long)n_ks);
  MIRL_REQUIRE(count_axis == MIRL_COUNT_ROWS || count_axis == MIRL_COUNT_K, "invalid count axis %d",
               count_axis);
  MIRL_REQUIRE(!accumulate || n_ks == 1, "accumulation takes one split");
  MIRL_REQUIRE(lda % 4 == 0 && ldb % 4 == 0 && lda >= K && ldb >= K,
               "row strides (%lld, %lld) must be multiples of 4 elements and >= K", (long long)lda,
               (long long)ldb);
  MIRL_REQUIRE((reinterpret_cast<uintptr_t>(A) & 15u) == 0 && (reinterpret_cast<uintptr_t>(B) & 15u) == 0,
               "operands must be 16-byte aligned");
  // buffer ranges of one 256-row tile are 32-bit byte counts
  MIRL_REQUIRE(kBM * lda * 4 < (int64_t(1) << 31) && kBN * ldb * 4 < (int64_t(1) << 31),
               "row strides (%lld, %lld) too large", (long long)lda, (long long)ldb);
  MIRL_REQUIRE(M < (int64_t(1) << 31) && N < (int64_t(1) << 31), "sizes exceed 2^31-1");
  MIRL_REQUIRE(ldc >= N, "output row stride %lld is smaller than N=%lld", (long long)ldc, (long long)N);
  LceParams P{};
  P.h = A;
  P.w = B;
  P.ldh = lda;
  P.ldw = ldb;
  P.V = N;
  P.Hd = K;
  P.row0 = 0;
  P.nrows = M;
  P.n_mt = ceil_div(M, kBM);
  P.n_nt = ceil_div(N, kBN);
  P.n_ks = n_ks;
  P.kb_len = kb;
  P.C = C;
  P.Cb = nullptr;
  P.ldc = ldc;
  P.accumulate = accumulate;
  P.count = count;
  P.count_off = count_off;
  P.count_axis = count_axis;
  P.final_at = 0;
  const int64_t grid = ceil_div(P.n_mt * P.n_nt * n_ks, kXcds) * kXcds;
  MIRL_REQUIRE(grid < (int64_t(1) << 31), "too many tiles");
  hipLaunchKernelGGL((lce_tile_kernel<kGemm, F32>), dim3((unsigned)grid), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), P);
  return check_launch("mirl_gemm_f32_abt");
}

extern "C" int mirl_lce_active_rows(const float* grad_out, int64_t g_stride_b, int64_t g_stride_s,
                                    int64_t T, int64_t bsz, const int64_t* target,
                                    int64_t t_stride_b, int64_t t_stride_s, const float* row_stats,
                                    const void* hidden, int dtype, int64_t Hd, int64_t ldh,
                                    int64_t* perm, int64_t* count, int64_t* target_out,
                                    float* stats_out, float* grad_rows, void* hidden_out,
                                    void* stream) {
  clear_error();
  MIRL_REQUIRE(lce_dtype_ok(dtype) || dtype == MIRL_DTYPE_F32,
               "hidden states must be bf16, fp16 or fp32 (dtype code %d)", dtype);
  MIRL_REQUIRE(T >= 0 && Hd > 0 && bsz > 0 && ldh >= Hd, "invalid shape T=%lld H=%lld B=%lld", (long long)T,
               (long long)Hd, (long long)bsz);
  MIRL_REQUIRE(T % bsz == 0, "row count %lld is not a multiple of the batch size %lld", (long long)T,
               (long long)bsz);
  MIRL_REQUIRE(T < (int64_t(1) << 31) - 8 * kActThreads, "too many rows (%lld)", (long long)T);
  MIRL_REQUIRE(count != nullptr, "null pointer argument");
  MIRL_REQUIRE(T == 0 || (grad_out && target && row_stats && hidden && perm && target_out && stats_out &&
                          grad_rows && hidden_out),
               "null pointer argument");
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(lce_active_rows_kernel, dim3(1), dim3(kActThreads), 0, st, grad_out, g_stride_b,
                     g_stride_s, (uint32_t)T, (uint32_t)bsz, perm, grad_rows, count);
  if (T > 0) {
    const int64_t esz = dtype == MIRL_DTYPE_F32 ? 4 : 2;
    const uintptr_t both = reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(hidden_out);
    auto launch = [&](auto unit) {
      using UNIT = decltype(unit);
      constexpr int64_t n = sizeof(UNIT);
      hipLaunchKernelGGL(lce_gather_rows_kernel<UNIT>, dim3((unsigned)std::min(T, kGatherGrid)), dim3(256), 0,
                         st, perm, count, T, (uint32_t)bsz, target, t_stride_b, t_stride_s, row_stats,
                         static_cast<const UNIT*>(hidden), Hd * esz / n, ldh * esz / n, target_out,
                         stats_out, static_cast<UNIT*>(hidden_out));
    };
    if ((both & 15u) == 0 && Hd * esz % 16 == 0 && ldh * esz % 16 == 0)
      launch(vu4{});
    else if (esz == 4)
      launch(uint32_t{});
    else
      launch(uint16_t{});
  }
  return check_launch("mirl_lce_active_rows");
}

extern "C" int mirl_transpose_f32(const float* src, int64_t R, int64_t C, int64_t lds, float* dst,
                                  int64_t ldd, int64_t R_pad, const int64_t* count, int64_t count_off,
                                  void* stream) {
  clear_error();
  MIRL_REQUIRE(R >= 0 && C >= 0 && R_pad >= R && lds >= C && ldd >= R_pad, "invalid shape");
  if (C == 0 || R_pad == 0) return MIRL_OK;
  MIRL_REQUIRE(src && dst, "null pointer argument");
  const int64_t n_rt = ceil_div(R_pad, 64), n_ct = ceil_div(C, 64);
  MIRL_REQUIRE(n_rt * n_ct < (int64_t(1) << 31), "too many tiles");
  hipLaunchKernelGGL(transpose_f32_kernel, dim3((unsigned)(n_rt * n_ct)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), src, R, C, lds, dst, ldd, R_pad, n_ct, count,
                     count_off);
  return check_launch("mirl_transpose_f32");
}
