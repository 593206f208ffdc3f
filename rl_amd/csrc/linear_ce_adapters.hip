// Token logprobs from hidden states and the output weight with low-rank adapters of several
// requests beside it, and their gradients.
//
//   d = dropout(h),  U = s_a (d . A_a^T),  x = h . W^T + U . B_a^T,  a the adapter of the row's sample
//   logprob_t = (x_t - m) - log(sum_v exp(x_v - m)),   G = (onehot(t) - softmax(x)) g
//   dU = s_a G . B_a,   dH = G . W + dropout'(dU . A_a),   dA_a = dU^T . d,   dB_a = G^T . U
//
// The [rows, V] logits are never written.  The rows are sorted by adapter, so a 256-row tile of
// the logits (lce_tile.h) meets few adapters; their part enters the tile's reduction as
// planes * r more hidden elements (U as two 16-bit values that add up to it; fp16: rows of U past
// its range from fp32 times a power of two, by themselves).  The logits stay fp32, and U, dU and
// their sums are fp32.
//
// Backward: the rows with a non-zero upstream gradient, sorted by adapter, in blocks.  Per block
// the tile loop writes G without its row factor g, in the operand type (fp16: times 2^15, which
// keeps probabilities down to 2^-40), and its transpose; dH = g (G . W) runs on the tile loop
// as well, and the adapters' three thin products on kernels of their own below, which are bound
// by reading G (dU), its transpose (dB) and the hidden states (dA) once.
//
// G is the one value on the way that is rounded to 16 bits: a gradient is then off by that
// rounding and its own (1.1 times the rounding of the result alone, measured), and G in fp32
// would double what dH's product reads.
//
// Step of 8 x 2048 tokens, 8200 of them active, 4 adapters of rank 16, H = 4096, V = 151936, bf16:
// 32 ms, of which the forward tiles 14.3, the gradient tiles 8.1 and dH 7.25 (1400 TFLOP/s, the
// library's product of the forward's operands 1495), dU 0.62 (2.5 GB of G, 4.0 TB/s), dB 0.49
// (5.1 TB/s), the down projection 0.11, dH's sum 0.08, dA 0.03.

#include "lce_tile.h"
#include "philox.h"

#pragma clang fp contract(off)

namespace mirl {
namespace {

constexpr int kRankTile = 64;  // ranks a kernel below handles together
constexpr float kF16Scale = 32768.f;

template <class E>
constexpr float g_scale_of() {
  return std::is_same<E, F16>::value ? kF16Scale : 1.f;
}

int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// A launch holds fewer than 2^32 threads.
constexpr int64_t kMaxRows = int64_t(1) << 26, kMaxBlocks = int64_t(1) << 23;
constexpr int64_t kMaxRank = 1024;  // a workgroup of adapter_dh_kernel holds its rows of dU in LDS
// Ranks of the plane arrays: whole tiles of those that with_rank chooses.
int64_t padded_rank(int64_t r8) { return r8 <= 16 ? 16 : r8 <= 32 ? 32 : round_up(r8, kRankTile); }

bool is16(int dtype) { return dtype == MIRL_DTYPE_BF16 || dtype == MIRL_DTYPE_F16; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// -------------------------------------------------------------------------------------------
// rows sorted by adapter
// -------------------------------------------------------------------------------------------
// Rows r = s * B + b, s < R.  A sample's key is its adapter + 1, or 0 for ids outside [0, N)
// (the base model).  The kept rows (all, or those with g != 0) go by key, then sample, then s.

__device__ __forceinline__ int64_t key_of(int64_t id, int64_t N) { return id >= 0 && id < N ? id + 1 : 0; }

// cnt[b] = kept rows of sample b.
__global__ __launch_bounds__(1024) void adapter_count_kernel(const float* __restrict__ g, int64_t gsb, int64_t gss,
                                                             int64_t R, int32_t* __restrict__ cnt) {
  __shared__ int w[16];
  const int64_t b = blockIdx.x;
  int n = 0;
  for (int64_t s = threadIdx.x; s < R; s += 1024) n += g[b * gsb + s * gss] != 0.f ? 1 : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int sum = 0;
    for (int i = 0; i < 16; ++i) sum += w[i];
    cnt[b] = sum;
  }
}

// Workgroup k: the samples of key k, in order.  start[b] = sorted place of sample b's first kept
// row; seg[a] that of adapter a's first row, seg[N] = *count = the rows kept.
__global__ __launch_bounds__(1024) void adapter_starts_kernel(const int64_t* __restrict__ ids, int64_t B, int64_t N,
                                                              int32_t R, const int32_t* __restrict__ cnt,
                                                              int32_t* __restrict__ start, int32_t* __restrict__ seg,
                                                              int64_t* __restrict__ count, int32_t* __restrict__ bad) {
  __shared__ int w[2][16];
  const int64_t k = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int before = 0;
  for (int64_t b = tid; b < B; b += 1024) before += key_of(ids[b], N) < k ? (cnt != nullptr ? cnt[b] : R) : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, kWave);
  if (lane == 0) w[0][wave] = before;
  __syncthreads();
  int at = 0;
  for (int i = 0; i < 16; ++i) at += w[0][i];
  if (tid == 0 && k > 0) {
    seg[k - 1] = at;
    if (bad != nullptr) bad[k - 1] = 0;
  }
  int turn = 1;
  for (int64_t b0 = 0; b0 < B; b0 += 1024) {
    const int64_t b = b0 + tid;
    const bool mine = b < B && key_of(ids[b], N) == k;
    const int n = mine ? (cnt != nullptr ? cnt[b] : R) : 0;
    int incl = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(incl, off, kWave);
      if (lane >= off) incl += o;
    }
    if (lane == 63) w[turn][wave] = incl;
    __syncthreads();  // the two buffers alternate: one barrier a round
    int pre = at;
    for (int i = 0; i < 16; ++i) {
      pre += i < wave ? w[turn][i] : 0;
      at += w[turn][i];
    }
    if (mine) start[b] = pre + incl - n;
    turn ^= 1;
  }
  if (tid == 0 && k == N) {
    seg[N] = at;
    *count = at;
  }
}

struct RowsOut {
  int64_t* perm;
  int32_t* aid;
  int64_t* target;
  float* g;      // or null
  float* stats;  // or null
};
// The kept rows of sample blockIdx.x: their original row, adapter, target, and for the backward
// their gradient and statistics.
__global__ __launch_bounds__(1024) void adapter_fill_kernel(const int64_t* __restrict__ ids, int64_t B, int64_t N,
                                                            int64_t R, const float* __restrict__ g, int64_t gsb,
                                                            int64_t gss, const int64_t* __restrict__ target,
                                                            int64_t tsb, int64_t tss, const float* __restrict__ stats,
                                                            const int32_t* __restrict__ start, RowsOut O) {
  __shared__ int w[2][16];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t aid = (int32_t)key_of(ids[b], N) - 1;
  int64_t at = start[b];
  int turn = 0;
  for (int64_t s0 = 0; s0 < R; s0 += 1024) {
    const int64_t s = s0 + tid;
    const float gv = g != nullptr && s < R ? g[b * gsb + s * gss] : 1.f;
    const bool keep = s < R && gv != 0.f;
    const uint64_t bal = __ballot(keep);
    if (lane == 0) w[turn][wave] = (int)__popcll(bal);
    __syncthreads();
    int64_t m = at + __popcll(bal & ((1ull << lane) - 1ull));
    for (int i = 0; i < 16; ++i) {
      m += i < wave ? w[turn][i] : 0;
      at += w[turn][i];
    }
    turn ^= 1;
    if (keep) {
      const int64_t r = s * B + b;
      O.perm[m] = r;
      O.aid[m] = aid;
      O.target[m] = target[b * tsb + s * tss];
      if (O.g != nullptr) O.g[m] = gv;
      if (O.stats != nullptr) {
        O.stats[2 * m] = stats[2 * r];
        O.stats[2 * m + 1] = stats[2 * r + 1];
      }
    }
  }
}

// -------------------------------------------------------------------------------------------
// small pieces shared by the kernels below
// -------------------------------------------------------------------------------------------
struct __attribute__((packed, aligned(2))) Raw8 {
  uint16_t e[8];
};
__device__ __forceinline__ vu4 zero4() { return vu4{0u, 0u, 0u, 0u}; }
// Eight 16-bit elements from p (any alignment).
__device__ __forceinline__ vu4 load_raw8(const uint16_t* p) {
  return __builtin_bit_cast(vu4, *reinterpret_cast<const Raw8*>(p));
}
// Elements c .. c + 7 of a row of H, zeros past its end.
__device__ __forceinline__ vu4 load_raw8_to(const uint16_t* row, int64_t c, int64_t H) {
  if (c + 8 <= H) return load_raw8(row + c);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = c + 2 * j < H ? row[c + 2 * j] : 0u, hi = c + 2 * j + 1 < H ? row[c + 2 * j + 1] : 0u;
    w[j] = lo | (hi << 16);
  }
  return vu4{w[0], w[1], w[2], w[3]};
}
// Elements whose bit of `keep` is clear become zero.
__device__ __forceinline__ vu4 mask8(vu4 q, uint32_t keep) {
  uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t m = ((keep >> (2 * j)) & 1u ? 0xffffu : 0u) | ((keep >> (2 * j)) & 2u ? 0xffff0000u : 0u);
    w[j] &= m;
  }
  return vu4{w[0], w[1], w[2], w[3]};
}
// Which of elements i .. i + 7 dropout keeps (any i).
__device__ __forceinline__ uint32_t keep8_at(uint64_t seed, const DropoutArgs& D, int64_t i) {
  const int sh = (int)(i & 7);
  const uint32_t a = dropout_keep8(seed, D.offset, (uint64_t)(i >> 3), D.threshold);
  if (sh == 0) return a;
  const uint32_t b = dropout_keep8(seed, D.offset, (uint64_t)(i >> 3) + 1, D.threshold);
  return ((a | (b << 8)) >> sh) & 0xffu;
}
template <class E>
__device__ __forceinline__ f32x4 mfma16(vu4 a, vu4 b, f32x4 c) {
  using frag = typename Mma<E>::frag;
  return Mma<E>::run(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c);
}
// v as kPlanes values of E that add up to it (to 2^-17 of it in bf16, 2^-23 in fp16 above its
// subnormal numbers).
template <class E>
__device__ __forceinline__ void split_planes(float v, uint16_t (&p)[kPlanes]) {
#pragma unroll
  for (int k = 0; k < kPlanes; ++k) {
    p[k] = bits_of<E>(v);
    v -= value_of<E>(p[k]);
  }
}

// -------------------------------------------------------------------------------------------
// forward: hidden rows gathered in sorted order, and U
// -------------------------------------------------------------------------------------------
struct DownParams {
  const uint16_t* hidden;  // [*, H], row stride ldh, original row order
  int64_t H, ldh;
  const int64_t* perm;
  const int32_t* aid;
  int64_t T;
  const uint16_t* A;       // [N, r, lda], zeros past H (lda a multiple of 8, 16-byte aligned)
  int64_t r, lda;
  const float* scaling;    // [N]
  DropoutArgs drop;
  uint16_t* h_out;         // [T, ldo], zeros in columns H .. ldo
  int64_t ldo;
  uint16_t* U;             // [T, kURow<E>, r8]
  int64_t r8;
  float* U32;              // [rows, r8] by original row, or null
  int64_t ny, nz;          // rank tiles, workgroups that share a row tile's adapters
  // and beside it, by workgroups past n_tiles * ny * nz: which adapters with rows hold an infinity or a
  // NaN in B ([N, b_vecs] 16-byte pieces, `per` workgroups an adapter)
  int64_t n_tiles;
  const vu4* B;
  int64_t b_vecs, per;
  const int32_t* seg;
  int32_t* bad;            // [N], zeros before: kBroken, and kWide from the rows themselves
};

constexpr int kScanVecs = 8;  // pieces a thread looks at
template <class E>
__device__ __forceinline__ void look_through(const DownParams& P, int64_t block) {
  const int64_t a = block / P.per, part = block - a * P.per;
  if (P.seg[a] >= P.seg[a + 1]) return;
  constexpr uint32_t ex = std::is_same<E, BF16>::value ? 0x7f80u : 0x7c00u;
  const vu4* src = P.B + a * P.b_vecs;
  vu4 q[kScanVecs];
#pragma unroll
  for (int u = 0; u < kScanVecs; ++u) {
    const int64_t i = (part * kScanVecs + u) * blockDim.x + threadIdx.x;
    q[u] = i < P.b_vecs ? src[i] : zero4();
  }
  bool none = false;
#pragma unroll
  for (int u = 0; u < kScanVecs; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) none |= (q[u][j] & ex) == ex || ((q[u][j] >> 16) & ex) == ex;
  if (none) atomicOr(P.bad + a, kBroken);
}

// 16 sorted rows a workgroup, the hidden dimension split over its NW waves 64 elements at a
// time.  An MFMA takes 16 ranks of the adapter against the 16 rows.  Rows of several adapters
// are read once per adapter (from the cache after the first time); the nz workgroups of the same
// rows take every nz-th adapter.
template <class E, int NT, int NW>
__global__ __launch_bounds__(NW * 64) void adapter_down_kernel(DownParams P) {
  __shared__ float red[NW][16][NT * 16 + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t shares = P.ny * P.nz;
  if ((int64_t)blockIdx.x >= P.n_tiles * shares) {
    look_through<E>(P, blockIdx.x - P.n_tiles * shares);
    return;
  }
  const int64_t tile = blockIdx.x / shares, share = blockIdx.x - tile * shares;
  const int by = (int)(share / P.nz), bz = (int)(share - by * P.nz);
  const int64_t m0 = tile * 16, rho0 = (int64_t)by * kRankTile;
  const int64_t m = m0 + lr;
  const bool live = m < P.T;
  const int64_t row = live ? P.perm[m] : 0;
  const int32_t my_aid = live ? P.aid[m] : -1;
  const uint16_t* hr = P.hidden + row * P.ldh;
  const uint64_t seed = P.drop.threshold > 0 ? P.drop.seed_of() : 0;
  if (share == 0) {
    uint16_t* ho = P.h_out + m * P.ldo;
#pragma unroll 4
    for (int64_t k0 = (int64_t)wave * 64; k0 < P.ldo; k0 += NW * 64) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t k = k0 + u * 32 + lg * 8;
        if (live && k < P.ldo) *reinterpret_cast<vu4*>(ho + k) = load_raw8_to(hr, k, P.H);
      }
    }
  }
  int done = -1;  // adapters up to this one are done (rows are sorted: ids ascend)
  for (int nth = 0;; ++nth) {
    // the smallest adapter of the 16 rows that is still to do
    int a = my_aid > done ? my_aid : 0x7fffffff;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
      const int o = __shfl_xor(a, off, kWave);
      a = o < a ? o : a;
    }
    a = __builtin_amdgcn_readfirstlane(a);
    if (a == 0x7fffffff) break;
    done = a;
    if (nth % (int)P.nz != bz) continue;
    const uint16_t* Aa = P.A + ((int64_t)a * P.r + rho0) * P.lda;
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const bool mine = my_aid == a;
    int64_t k0 = (int64_t)wave * 64;
    // two steps at a time while they end inside the row: their loads in flight together
    constexpr int KU = NT < 4 ? 4 : 2;
    for (; k0 + (KU / 2 - 1) * NW * 64 + 64 <= P.H; k0 += KU / 2 * NW * 64) {
      vu4 h[KU], w[KU][NT];
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int64_t k = k0 + (u / 2) * NW * 64 + (u & 1) * 32 + lg * 8;
        h[u] = mine ? load_raw8(hr + k) : zero4();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int64_t rho = t * 16 + lr;
          w[u][t] = rho0 + rho < P.r ? *reinterpret_cast<const vu4*>(Aa + rho * P.lda + k) : zero4();
        }
      }
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int64_t k = k0 + (u / 2) * NW * 64 + (u & 1) * 32 + lg * 8;
        if (P.drop.threshold > 0) h[u] = mask8(h[u], keep8_at(seed, P.drop, row * P.H + k));
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = mfma16<E>(w[u][t], h[u], acc[t]);
      }
    }
    for (; k0 < P.H; k0 += NW * 64) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t k = k0 + u * 32 + lg * 8;
        vu4 h = mine && k < P.H ? load_raw8_to(hr, k, P.H) : zero4();
        if (P.drop.threshold > 0) h = mask8(h, keep8_at(seed, P.drop, row * P.H + k));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int64_t rho = t * 16 + lr;
          const vu4 w = rho0 + rho < P.r && k < P.H ? *reinterpret_cast<const vu4*>(Aa + rho * P.lda + k) : zero4();
          acc[t] = mfma16<E>(w, h, acc[t]);
        }
      }
    }
    // acc[t][e] of a lane: rank t * 16 + lg * 4 + e of row lr
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][lr][t * 16 + lg * 4 + e] = acc[t][e];
    __syncthreads();
    const float s = P.scaling[a] * (P.drop.threshold > 0 ? P.drop.scale : 1.f);
    for (int q = tid; q < 16 * NT * 16; q += NW * 64) {
      const int rl = q / (NT * 16), rho = q - rl * (NT * 16);
      const int64_t mm = m0 + rl;
      if (mm >= P.T || P.aid[mm] != a || rho0 + rho >= P.r8) continue;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) v += red[i][rl][rho];
      v *= s;
      if constexpr (std::is_same<E, F16>::value) {
        const uint32_t mag = __float_as_uint(v) & 0x7fffffffu;
        if (mag >= kF16Past && mag < 0x7f800000u) atomicOr(P.bad + a, kWide);  // (its planes are not used)
        u_f32(P.U, mm, (int)P.r8)[rho0 + rho] = v;
      }
      uint16_t p[kPlanes];
      split_planes<E>(v, p);
#pragma unroll
      for (int k = 0; k < kPlanes; ++k) P.U[(mm * kURow<E> + k) * P.r8 + rho0 + rho] = p[k];
      if (P.U32 != nullptr) P.U32[P.perm[mm] * P.r8 + rho0 + rho] = v;
    }
    __syncthreads();
  }
}

// -------------------------------------------------------------------------------------------
// backward: the active rows' operands
// -------------------------------------------------------------------------------------------
// Row m < *count: its hidden row (zero padded to ldo) and the planes of its U.
template <class E>
__global__ __launch_bounds__(256) void adapter_gather_kernel(const int64_t* __restrict__ perm,
                                                             const int32_t* __restrict__ aid,
                                                             const int64_t* __restrict__ count,
                                                             const uint16_t* __restrict__ hidden, int64_t H,
                                                             int64_t ldh, const float* __restrict__ U32, int64_t r8,
                                                             uint16_t* __restrict__ h_out, int64_t ldo,
                                                             uint16_t* __restrict__ U) {
  const int64_t n = *count;
  for (int64_t m = blockIdx.x; m < n; m += gridDim.x) {
    const int64_t row = perm[m];
    const uint16_t* hr = hidden + row * ldh;
    for (int64_t k = (int64_t)threadIdx.x * 8; k < ldo; k += 256 * 8)
      *reinterpret_cast<vu4*>(h_out + m * ldo + k) = load_raw8_to(hr, k, H);
    if (aid[m] < 0) continue;
    for (int64_t rho = threadIdx.x; rho < r8; rho += 256) {
      const float v = U32[row * r8 + rho];
      uint16_t p[kPlanes];
      split_planes<E>(v, p);
#pragma unroll
      for (int k = 0; k < kPlanes; ++k) U[(m * kURow<E> + k) * r8 + rho] = p[k];
      if constexpr (std::is_same<E, F16>::value) u_f32(U, m, (int)r8)[rho] = v;
    }
  }
}

// dst[z][c][r] = src[z][r][c] (16-bit elements) for r < R (R lowered to *count with one),
// zeros for R <= r < Rp; with `perm` row r's elements are dropped as those of original row
// perm[r].  64 x 64 tiles through LDS; with a count, tiles past the one that holds the last row
// are left as they were.
struct TransposeParams {
  const uint16_t* src;
  int64_t R, C, lds, src_z;
  uint16_t* dst;
  int64_t ldd, Rp, dst_z;
  int64_t n_ct, n_rt;
  const int64_t* count;
  const int64_t* perm;
  DropoutArgs drop;
};
__global__ __launch_bounds__(256) void adapter_transpose_kernel(TransposeParams P) {
  constexpr int kP = 66;  // row pitch: the rows that a wave's column read touches start in different banks
  __shared__ uint16_t tile[64 * kP];
  int64_t R = P.R;
  if (P.count != nullptr && *P.count < R) R = *P.count;
  const int64_t z = blockIdx.x / (P.n_ct * P.n_rt), in = blockIdx.x - z * (P.n_ct * P.n_rt);
  const int64_t tr = in / P.n_ct, tc = in - tr * P.n_ct;
  const int64_t r0 = tr * 64, c0 = tc * 64;
  if (P.count != nullptr && r0 >= R) return;
  const uint16_t* src = P.src + z * P.src_z;
  uint16_t* dst = P.dst + z * P.dst_z;
  const bool drop = P.perm != nullptr && P.drop.threshold > 0;
  const uint64_t seed = drop ? P.drop.seed_of() : 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int idx = (int)threadIdx.x + 256 * k, lr = idx >> 3, cg = (idx & 7) * 8;
    const int64_t r = r0 + lr, c = c0 + cg;
    vu4 q = zero4();
    if (r < R && c < P.C) {
      q = load_raw8_to(src + r * P.lds, c, P.C);
      if (drop) q = mask8(q, keep8_at(seed, P.drop, P.perm[r] * P.C + c));
    }
    uint32_t* t32 = reinterpret_cast<uint32_t*>(tile + lr * kP + cg);
    t32[0] = q.x;
    t32[1] = q.y;
    t32[2] = q.z;
    t32[3] = q.w;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int idx = (int)threadIdx.x + 256 * k, lc = idx >> 3, rg = (idx & 7) * 8;
    const int64_t c = c0 + lc, r = r0 + rg;
    if (c >= P.C || r >= P.Rp) continue;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = (uint32_t)tile[(rg + 2 * j) * kP + lc] | ((uint32_t)tile[(rg + 2 * j + 1) * kP + lc] << 16);
    // (Rp and ldd are multiples of 8, dst 16-byte aligned)
    *reinterpret_cast<vu4*>(dst + c * P.ldd + r) = vu4{w[0], w[1], w[2], w[3]};
  }
}

// -------------------------------------------------------------------------------------------
// backward of one block: sorted rows row0 .. row0 + n (as far as *count)
// -------------------------------------------------------------------------------------------
struct BlockParams {
  int64_t row0, n;
  const int64_t* count;
  const int64_t* perm;
  const int32_t* aid;
  const int32_t* seg;
  int64_t N, V, H, r, r8;
  const float* g;          // [rows] of the sorted rows
  const float* scaling;    // [N]
  const uint16_t* G;       // [n, ldg] of the operand type, without g, times g_scale
  int64_t ldg;
  const uint16_t* Gt;      // [V, ldgt]
  int64_t ldgt;
  const uint16_t* BT;      // [N, r8, ldbt]: B transposed, zeros past V
  int64_t ldbt;
  const uint16_t* A;       // [N, r, lda]
  int64_t lda;
  const uint16_t* hT;      // [H, ldht]: the dropped hidden rows, transposed
  int64_t ldht;
  const float* U32;        // [rows, r8] by original row
  DropoutArgs drop;
  int64_t splits, k_len;   // dU's split of the vocabulary
  float* du_part;          // [splits, n, r8]
  float* du;               // [n, r8]: dU with s_a and g
  uint32_t* peak;          // [n, 2]: an adapter's largest |dU| and |g U| (fp16), as bits, at its first row (peak_of)
  uint16_t* duT;           // [kPlanes, r16, ldn]: dU transposed, scaled into range (fp16)
  uint16_t* ugT;           // [kPlanes, r16, ldn]: g U transposed, likewise
  int64_t ldn, r16;
  const float* h_part;     // [h_splits, n, H]: G . W
  int64_t h_splits;
  void* dH;                // [*, H] by original row
  int64_t lddh;
  float* dA;               // [N, r, H]
  float* dB;               // [N, V, r]
};

__device__ __forceinline__ int64_t block_rows(const BlockParams& P) {
  const int64_t c = *P.count - P.row0;
  return c < 0 ? 0 : c < P.n ? c : P.n;
}

// An adapter's maxima in the block: at the place of its first row there.
__device__ __forceinline__ uint32_t* peak_of(const BlockParams& P, int64_t a) {
  const int64_t first = P.seg[a] - P.row0;
  return P.peak + 2 * (first > 0 ? first : 0);
}

// dU's partial sums: a wave takes 32 rows and a range of the vocabulary, once per adapter
// among its rows.  (Also clears the maxima that the next kernel takes.)
template <class E, int NT>
__global__ __launch_bounds__(256) void adapter_du_kernel(BlockParams P) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t n = block_rows(P);
  const int64_t n_rt = (P.n + 127) / 128;
  const int64_t split = blockIdx.x / n_rt, rt = blockIdx.x - split * n_rt;
  const int64_t w0 = rt * 128 + wave * 32, rho0 = (int64_t)blockIdx.y * kRankTile;
  if (std::is_same<E, F16>::value && split == 0 && blockIdx.y == 0) {
    const int64_t m = rt * 128 + (tid >> 1);
    if (m < n) P.peak[2 * m + (tid & 1)] = 0;
  }
  if (w0 >= n) return;
  const int64_t w1 = w0 + 32 < n ? w0 + 32 : n;
  const int64_t k_end = (split + 1) * P.k_len < P.ldbt ? (split + 1) * P.k_len : P.ldbt;
  int64_t cur = w0;
  while (cur < w1) {
    const int a = __builtin_amdgcn_readfirstlane(P.aid[P.row0 + cur]);
    // the rows of this adapter end where the next one's begin (none: where the first one's do)
    const int64_t next_seg = P.seg[a + 1] - P.row0;
    const int64_t next = next_seg < w1 ? next_seg : w1;
    if (a >= 0) {
      const uint16_t* Ba = P.BT + ((int64_t)a * P.r8 + rho0) * P.ldbt;
      f32x4 acc[2][NT];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      // rows past the block's are read as its last one
      const int64_t ra = w0 + lr < n ? w0 + lr : n - 1, rb = w0 + 16 + lr < n ? w0 + 16 + lr : n - 1;
      const uint16_t *ga = P.G + ra * P.ldg, *gb = P.G + rb * P.ldg;
      // KU steps of 32 columns at a time, their loads in flight together (k_len and the rows'
      // padded length are multiples of 128)
      constexpr int KU = NT < 4 ? 4 : 2;
      for (int64_t k0 = split * P.k_len; k0 < k_end; k0 += KU * 32) {
        vu4 q0[KU], q1[KU], b[KU][NT];
#pragma unroll
        for (int u = 0; u < KU; ++u) {
          const int64_t k = k0 + u * 32 + lg * 8;
          q0[u] = *reinterpret_cast<const vu4*>(ga + k);
          q1[u] = *reinterpret_cast<const vu4*>(gb + k);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const int64_t rho = t * 16 + lr;
            b[u][t] = rho0 + rho < P.r8 ? *reinterpret_cast<const vu4*>(Ba + rho * P.ldbt + k) : zero4();
          }
        }
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[0][t] = mfma16<E>(b[u][t], q0[u], acc[0][t]);
            acc[1][t] = mfma16<E>(b[u][t], q1[u], acc[1][t]);
          }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t m = w0 + i * 16 + lr;
        if (m < cur || m >= next) continue;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int64_t rho = rho0 + t * 16 + lg * 4;
          if (rho < P.r8) *reinterpret_cast<f32x4*>(P.du_part + (split * P.n + m) * P.r8 + rho) = acc[i][t];
        }
      }
    }
    cur = next;
  }
}

// dU = s_a g (sum of the splits), in split order; each adapter's largest magnitudes of dU and g U.
template <class E>
__global__ __launch_bounds__(256) void adapter_du_sum_kernel(BlockParams P) {
  const int64_t n = block_rows(P), total = n * P.r8;
  const int lane = threadIdx.x & 63;
  // (whole waves go round: 64 elements each)
  for (int64_t i0 = (int64_t)blockIdx.x * 256 + (threadIdx.x & ~63); i0 < total; i0 += (int64_t)gridDim.x * 256) {
    const int64_t i = i0 + lane;
    int32_t a = -1;
    uint32_t pu = 0, pg = 0;
    if (i < total) {
      const int64_t m = i / P.r8, rho = i - m * P.r8;
      a = P.aid[P.row0 + m];
      float v = 0.f;
      const float g = P.g[P.row0 + m];
      if (a >= 0) {
#pragma unroll 8
        for (int64_t s = 0; s < P.splits; ++s) v += P.du_part[(s * P.n + m) * P.r8 + rho];
        v *= (1.f / g_scale_of<E>()) * P.scaling[a];
        v *= g;
        const uint32_t b = __float_as_uint(g * P.U32[P.perm[P.row0 + m] * P.r8 + rho]) & 0x7fffffffu;
        const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
        // (values that are none do not set the scale)
        pu = u < 0x7f800000u ? u : 0u;
        pg = b < 0x7f800000u ? b : 0u;
      }
      P.du[i] = v;
    }
    if constexpr (std::is_same<E, F16>::value) {
      uint64_t todo = __ballot(a >= 0);
      while (todo != 0) {  // the adapters of the wave's rows, one after the other
        const int32_t at = __shfl(a, __ffsll((unsigned long long)todo) - 1, kWave);
        const bool mine = a == at;
        uint32_t mu = mine ? pu : 0u, mg = mine ? pg : 0u;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
          const uint32_t x = (uint32_t)__shfl_xor((int)mu, off, kWave), y = (uint32_t)__shfl_xor((int)mg, off, kWave);
          mu = x > mu ? x : mu;
          mg = y > mg ? y : mg;
        }
        if (lane == 0) {
          uint32_t* peak = peak_of(P, at);
          atomicMax(peak, mu);  // maxima of whole numbers: any order gives the same
          atomicMax(peak + 1, mg);
        }
        todo &= ~__ballot(mine);
      }
    }
  }
}

// The power of two that takes the largest magnitude (its bits) to [2^14, 2^15), for fp16
// planes; 1 for bf16, which has fp32's range, and for zeros.
template <class E>
__device__ __forceinline__ float plane_scale(const uint32_t* peak) {
  if constexpr (!std::is_same<E, F16>::value) return 1.f;
  const int e = (int)(*peak >> 23);
  if (e == 0) return 1.f;
  int up = 14 + 127 - e;
  up = up > 120 ? 120 : up < -120 ? -120 : up;
  return __uint_as_float((uint32_t)(127 + up) << 23);
}

// dU and g U as planes, transposed: columns m < n, zeros up to ldn and in ranks past r.
template <class E>
__global__ __launch_bounds__(256) void adapter_planes_kernel(BlockParams P) {
  const int64_t n = block_rows(P);
  const int64_t width = (n + 63) / 64 * 64;  // what the products below read
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < width * P.r16; i += (int64_t)gridDim.x * 256) {
    const int64_t rho = i / width, m = i - rho * width;
    float u = 0.f, gu = 0.f;
    const int32_t a = m < n && rho < P.r8 ? P.aid[P.row0 + m] : -1;
    if (a >= 0) {
      const uint32_t* peak = peak_of(P, a);
      u = P.du[m * P.r8 + rho] * plane_scale<E>(peak);
      gu = (P.g[P.row0 + m] * P.U32[P.perm[P.row0 + m] * P.r8 + rho]) * plane_scale<E>(peak + 1);
    }
    uint16_t pu[kPlanes], pg[kPlanes];
    split_planes<E>(u, pu);
    split_planes<E>(gu, pg);
#pragma unroll
    for (int k = 0; k < kPlanes; ++k) {
      P.duT[(k * P.r16 + rho) * P.ldn + m] = pu[k];
      P.ugT[(k * P.r16 + rho) * P.ldn + m] = pg[k];
    }
  }
}

// Bits of the eight elements m .. m + 7 that lie in [lo, hi).
__device__ __forceinline__ uint32_t inside8(int64_t m, int64_t lo, int64_t hi) {
  const int64_t a = lo - m, b = hi - m;
  const uint32_t from = a <= 0 ? 0xffu : a >= 8 ? 0u : (0xffu << a) & 0xffu;
  const uint32_t to = b >= 8 ? 0xffu : b <= 0 ? 0u : 0xffu >> (8 - b);
  return from & to;
}

// 64 columns from k0 on of the product below; those outside [lo, hi) are zero in both operands (a
// row of another adapter may hold infinities or NaN).
template <class E, int NT, int MT>
__device__ __forceinline__ void thin_piece(const uint16_t* const (&x)[MT], const uint16_t* y, int64_t plane,
                                           int64_t ldn, int64_t k0, int64_t lo, int64_t hi, int lg,
                                           f32x4 (&acc)[MT][NT]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t k = k0 + u * 32 + lg * 8;
    const uint32_t in = inside8(k, lo, hi);
    vu4 q[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) q[i] = mask8(*reinterpret_cast<const vu4*>(x[i] + k), in);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int p = 0; p < kPlanes; ++p) {
        const vu4 b = mask8(*reinterpret_cast<const vu4*>(y + p * plane + (int64_t)t * 16 * ldn + k), in);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][t] = mfma16<E>(q[i], b, acc[i][t]);
      }
  }
}

// MT 16-row tiles of X against the planes Y [kPlanes, r16, ldn], summed over the columns [lo, hi)
// in pieces of 64 from k0 on, every step-th column.
template <class E, int NT, int MT>
__device__ __forceinline__ void thin_product(const uint16_t* const (&x)[MT], const uint16_t* y, int64_t plane,
                                             int64_t ldn, int64_t k0, int64_t step, int64_t lo, int64_t hi, int lg,
                                             f32x4 (&acc)[MT][NT]) {
  // whole pieces two at a time, their loads in flight together
  while (k0 < lo) {
    thin_piece<E, NT, MT>(x, y, plane, ldn, k0, lo, hi, lg, acc);
    k0 += step;
  }
  for (; k0 + step + 64 <= hi; k0 += 2 * step) {
    vu4 q[4][MT], b[4][NT][kPlanes];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t k = k0 + (u >> 1) * step + (u & 1) * 32 + lg * 8;
#pragma unroll
      for (int i = 0; i < MT; ++i) q[u][i] = *reinterpret_cast<const vu4*>(x[i] + k);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int p = 0; p < kPlanes; ++p)
          b[u][t][p] = *reinterpret_cast<const vu4*>(y + p * plane + (int64_t)t * 16 * ldn + k);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int p = 0; p < kPlanes; ++p)
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][t] = mfma16<E>(q[u][i], b[u][t][p], acc[i][t]);
  }
  for (; k0 < hi; k0 += step) thin_piece<E, NT, MT>(x, y, plane, ldn, k0, lo, hi, lg, acc);
}

// dB_a += G^T . (g U): 32 vocabulary rows a wave, once per adapter with rows in the block; with
// few vocabulary rows gridDim.z workgroups share their adapters.
template <class E, int NT>
__global__ __launch_bounds__(256) void adapter_db_kernel(BlockParams P) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t n = block_rows(P);
  const int64_t v0 = ((int64_t)blockIdx.x * 4 + wave) * 32, rho0 = (int64_t)blockIdx.y * kRankTile;
  if (v0 >= P.V || n == 0) return;
  const uint16_t* x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) x[i] = P.Gt + (v0 + i * 16 + lr < P.V ? v0 + i * 16 + lr : P.V - 1) * P.ldgt;
  const uint16_t* y = P.ugT + (rho0 + lr) * P.ldn;
  int64_t a = P.aid[P.row0] < 0 ? 0 : P.aid[P.row0];
  const int64_t a_last = P.aid[P.row0 + n - 1];
  unsigned nth = 0;
  for (; a <= a_last; ++a) {
    int64_t lo = P.seg[a] - P.row0, hi = P.seg[a + 1] - P.row0;
    lo = lo < 0 ? 0 : lo;
    hi = hi > n ? n : hi;
    if (lo >= hi || nth++ % gridDim.z != blockIdx.z) continue;
    f32x4 acc[2][NT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float scale = 1.f / (plane_scale<E>(P.peak + 2 * lo + 1) * g_scale_of<E>());
    thin_product<E, NT, 2>(x, y, P.r16 * P.ldn, P.ldn, lo / 64 * 64, 64, lo, hi, lg, acc);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t v = v0 + i * 16 + lg * 4 + e;
        if (v >= P.V) continue;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int64_t rho = rho0 + t * 16 + lr;
          if (rho < P.r) P.dB[(a * P.V + v) * P.r + rho] += acc[i][t][e] * scale;
        }
      }
  }
}

// dA_a += dU^T . d: 16 hidden columns a workgroup, the rows split over its 16 waves.
constexpr int kDaWaves = 16;
template <class E, int NT>
__global__ __launch_bounds__(kDaWaves * 64) void adapter_da_kernel(BlockParams P) {
  __shared__ float red[kDaWaves][16][NT * 16 + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t n = block_rows(P);
  if (n == 0) return;
  const int64_t h0 = (int64_t)blockIdx.x * 16, rho0 = (int64_t)blockIdx.y * kRankTile;
  const uint16_t* x[1] = {P.hT + (h0 + lr < P.H ? h0 + lr : P.H - 1) * P.ldht + P.row0};
  const uint16_t* y = P.duT + (rho0 + lr) * P.ldn;
  int64_t a = P.aid[P.row0] < 0 ? 0 : P.aid[P.row0];
  const int64_t a_last = P.aid[P.row0 + n - 1];
  for (; a <= a_last; ++a) {
    int64_t lo = P.seg[a] - P.row0, hi = P.seg[a + 1] - P.row0;
    lo = lo < 0 ? 0 : lo;
    hi = hi > n ? n : hi;
    if (lo >= hi) continue;
    f32x4 acc[1][NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float scale = (P.drop.threshold > 0 ? P.drop.scale : 1.f) / plane_scale<E>(P.peak + 2 * lo);
    thin_product<E, NT, 1>(x, y, P.r16 * P.ldn, P.ldn, lo / 64 * 64 + wave * 64, kDaWaves * 64, lo, hi, lg, acc);
    __syncthreads();  // the last adapter's sums are read
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][lg * 4 + e][t * 16 + lr] = acc[0][t][e];
    __syncthreads();
    for (int q = tid; q < 16 * NT * 16; q += kDaWaves * 64) {
      const int hl = q & 15, rho = q >> 4;
      if (h0 + hl >= P.H || rho0 + rho >= P.r) continue;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kDaWaves; ++w) v += red[w][hl][rho];
      P.dA[(a * P.r + rho0 + rho) * P.H + h0 + hl] += v * scale;
    }
  }
}

// dH of the block's rows: g (sum of the splits of G . W) + dropout'(dU . A_a), rounded once.  ROWS
// rows a workgroup, eight columns a thread; the rows' adapters one after the other.
constexpr int kDhRows = 4;
template <class E, int ROWS>
__global__ __launch_bounds__(256) void adapter_dh_kernel(BlockParams P) {
  extern __shared__ float du_s[];  // [ROWS][r8]
  const int64_t n = block_rows(P);
  const int64_t n_ct = (P.H + 2047) / 2048;
  const int64_t rt = blockIdx.x / n_ct, ct = blockIdx.x - rt * n_ct;
  const int64_t m0 = rt * ROWS, c = (ct * 256 + threadIdx.x) * 8;
  if (m0 >= n) return;
  const int rows = n - m0 < ROWS ? (int)(n - m0) : ROWS;
  for (int q = threadIdx.x; q < rows * (int)P.r8; q += 256) du_s[q] = P.du[m0 * P.r8 + q];
  __syncthreads();
  if (c >= P.H) return;
  const bool full = c + 8 <= P.H;
  float add[ROWS][8];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) add[i][e] = 0.f;
  int cur = 0;
  while (cur < rows) {
    const int a = P.aid[P.row0 + m0 + cur];
    const int64_t end = P.seg[a + 1] - P.row0 - m0;
    const int next = end < rows ? (int)end : rows;
    if (a >= 0) {
      const uint16_t* Aa = P.A + (int64_t)a * P.r * P.lda;
      // four ranks at a time, their loads in flight together (r8 holds a multiple of eight)
      for (int64_t rho = 0; rho < P.r; rho += 4) {
        vu4 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = rho + j < P.r ? load_raw8_to(Aa + (rho + j) * P.lda, c, P.H) : zero4();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float w[8];
          E::unpack(q[j], w);
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            if (i < cur || i >= next) continue;
            const float d = du_s[i * P.r8 + rho + j];
#pragma unroll
            for (int e = 0; e < 8; ++e) add[i][e] = fmaf(d, w[e], add[i][e]);
          }
        }
      }
    }
    cur = next;
  }
  const uint64_t seed = P.drop.threshold > 0 ? P.drop.seed_of() : 0;
  // the splits' sums of all rows, their loads in flight together (rows past the block's end
  // read its last one)
  float sum[ROWS][8];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[i][e] = 0.f;
  const bool vec = full && P.H % 4 == 0;
  constexpr int kU = ROWS == 1 ? 4 : 1;
#pragma unroll kU
  for (int64_t s = 0; s < P.h_splits; ++s) {
    const float* src = P.h_part + (s * P.n + m0) * P.H + c;
    if (vec) {
      float4 q[ROWS][2];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float4* row = reinterpret_cast<const float4*>(src + (i < rows ? i : rows - 1) * P.H);
        q[i][0] = row[0];
        q[i][1] = row[1];
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        sum[i][0] += q[i][0].x; sum[i][1] += q[i][0].y; sum[i][2] += q[i][0].z; sum[i][3] += q[i][0].w;
        sum[i][4] += q[i][1].x; sum[i][5] += q[i][1].y; sum[i][6] += q[i][1].z; sum[i][7] += q[i][1].w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i < rows && c + e < P.H) sum[i][e] += src[i * P.H + e];
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (i >= rows) break;
    const int64_t m = m0 + i, row = P.perm[P.row0 + m];
    const float g = P.g[P.row0 + m] * (1.f / g_scale_of<E>());
    float (&o)[8] = sum[i];
    uint32_t keep = 0xffu;
    float ds = 1.f;
    if (P.drop.threshold > 0) {
      keep = keep8_at(seed, P.drop, row * P.H + c);
      ds = P.drop.scale;
    }
    const bool adapted = P.aid[P.row0 + m] >= 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[e] *= g;
      if (adapted && ((keep >> e) & 1u)) o[e] = fmaf(add[i][e], ds, o[e]);
    }
    uint16_t* dst = static_cast<uint16_t*>(P.dH) + row * P.lddh + c;
    if (full && P.H % 8 == 0) {
      *reinterpret_cast<vu4*>(dst) = E::pack(o);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < P.H) dst[e] = bits_of<E>(o[e]);
    }
  }
}

// f(E, NT) for the operand type and the rank tiles of min(r, 64) ranks.
template <class F>
void with_rank(int dtype, int64_t r8, F&& f) {
  auto go = [&](auto e) {
    if (r8 <= 16)
      f(e, std::integral_constant<int, 1>{});
    else if (r8 <= 32)
      f(e, std::integral_constant<int, 2>{});
    else
      f(e, std::integral_constant<int, 4>{});
  };
  if (dtype == MIRL_DTYPE_BF16)
    go(BF16{});
  else
    go(F16{});
}

int check_operands(int dtype, const void* hidden, int64_t Hd, int64_t ldh, const void* weight, int64_t V, int64_t ldw) {
  MIRL_REQUIRE(is16(dtype), "hidden states, weight and adapters must be bf16 or fp16 (dtype code %d)", dtype);
  MIRL_REQUIRE(V > 0 && Hd > 0 && V < (int64_t(1) << 31), "invalid shape V=%lld H=%lld", (long long)V, (long long)Hd);
  MIRL_REQUIRE(Hd % 8 == 0 && ldh % 8 == 0 && ldw % 8 == 0 && ldh >= padded_hidden(Hd, 2) && ldw >= Hd &&
                   ldh < (int64_t(1) << 22) && ldw < (int64_t(1) << 22),
               "hidden size %lld and row strides (%lld, %lld) must be multiples of 8, the hidden states' rows padded to %lld, "
               "and the strides below 2^22",
               (long long)Hd, (long long)ldh, (long long)ldw, (long long)padded_hidden(Hd, 2));
  MIRL_REQUIRE(aligned16(hidden) && aligned16(weight), "hidden states and weight must be 16-byte aligned");
  return MIRL_OK;
}

}  // namespace
}  // namespace mirl

using namespace mirl;

extern "C" int mirl_adapter_rows(const int64_t* ids, int64_t B, int64_t N, int64_t R, const float* grad_out,
                                 int64_t g_stride_b, int64_t g_stride_s, const int64_t* target, int64_t t_stride_b,
                                 int64_t t_stride_s, const float* row_stats, int64_t* perm, int32_t* adapter,
                                 int64_t* target_out, float* grad_rows, float* stats_out, int32_t* seg, int64_t* count,
                                 int32_t* bad, int32_t* workspace, void* stream) {
  clear_error();
  MIRL_REQUIRE(B > 0 && N > 0 && R > 0, "invalid shape B=%lld N=%lld R=%lld", (long long)B, (long long)N, (long long)R);
  MIRL_REQUIRE(B < (int64_t(1) << 22) && N < (int64_t(1) << 22) && R < kMaxRows && B * R < kMaxRows,
               "sizes reach 2^26 rows, 2^22 samples or 2^22 adapters");
  MIRL_REQUIRE(ids && target && perm && adapter && target_out && seg && count && workspace, "null pointer argument");
  MIRL_REQUIRE((row_stats == nullptr) == (stats_out == nullptr) && (grad_out == nullptr) == (grad_rows == nullptr),
               "null pointer argument");
  hipStream_t st = static_cast<hipStream_t>(stream);
  int32_t *cnt = workspace, *start = workspace + B;
  if (grad_out != nullptr)
    hipLaunchKernelGGL(adapter_count_kernel, dim3((unsigned)B), dim3(1024), 0, st, grad_out, g_stride_b, g_stride_s, R, cnt);
  hipLaunchKernelGGL(adapter_starts_kernel, dim3((unsigned)(N + 1)), dim3(1024), 0, st, ids, B, N, (int32_t)R,
                     grad_out != nullptr ? cnt : nullptr, start, seg, count, bad);
  hipLaunchKernelGGL(adapter_fill_kernel, dim3((unsigned)B), dim3(1024), 0, st, ids, B, N, R, grad_out, g_stride_b,
                     g_stride_s, target, t_stride_b, t_stride_s, row_stats, start,
                     RowsOut{perm, adapter, target_out, grad_rows, stats_out});
  return check_launch("mirl_adapter_rows");
}

extern "C" int mirl_adapter_down(const void* hidden, int dtype, int64_t Hd, int64_t ldh, const int64_t* perm,
                                 const int32_t* adapter, int64_t T, const void* a, int64_t N, int64_t r, int64_t lda, const float* scaling,
                                 double p, int64_t seed, const int64_t* seed_dev, int64_t offset, void* hidden_out,
                                 int64_t ldo, void* u_planes, int64_t r8, float* u_rows, const void* b,
                                 int64_t b_elems, const int32_t* seg, int32_t* bad, void* stream) {
  clear_error();
  MIRL_REQUIRE(is16(dtype), "hidden states and adapters must be bf16 or fp16 (dtype code %d)", dtype);
  MIRL_REQUIRE(T > 0 && T < kMaxRows && Hd > 0 && N > 0 && r > 0 && r8 >= r && r8 % 8 == 0 && r8 <= kMaxRank && ldh >= Hd &&
                   ldo >= Hd && ldo % 8 == 0,
               "invalid shape T=%lld H=%lld r=%lld r8=%lld ldo=%lld", (long long)T, (long long)Hd, (long long)r,
               (long long)r8, (long long)ldo);
  MIRL_REQUIRE(p >= 0.0 && p <= 1.0, "dropout probability %g is outside [0, 1]", p);
  MIRL_REQUIRE(hidden && perm && adapter && a && scaling && hidden_out && u_planes && b && seg && bad,
               "null pointer argument");
  MIRL_REQUIRE(b_elems > 0 && b_elems % 8 == 0 && aligned16(b), "adapters of %lld elements", (long long)b_elems);
  MIRL_REQUIRE(lda >= Hd && lda % 8 == 0 && aligned16(a) && aligned16(hidden_out) && aligned16(u_planes),
               "the adapters' rows must be 16-byte aligned (row stride %lld)", (long long)lda);
  // few rows: 16 waves share them, and workgroups their adapters, to have the loads of all in
  // flight (64 rows of 16 adapters, H = 4096: 91 -> 18 us, 23 with the look at 78 MB of B beside
  // it); many: four waves (108 us of [16384, 4096])
  const bool few = T <= 2048;
  DownParams P{};
  P.hidden = static_cast<const uint16_t*>(hidden);
  P.H = Hd;
  P.ldh = ldh;
  P.perm = perm;
  P.aid = adapter;
  P.T = T;
  P.A = static_cast<const uint16_t*>(a);
  P.r = r;
  P.lda = lda;
  P.scaling = scaling;
  P.drop = dropout_args(p, seed, seed_dev, offset);
  P.h_out = static_cast<uint16_t*>(hidden_out);
  P.ldo = ldo;
  P.U = static_cast<uint16_t*>(u_planes);
  P.r8 = r8;
  P.U32 = u_rows;
  P.n_tiles = ceil_div(T, 16);
  P.B = static_cast<const vu4*>(b);
  P.b_vecs = b_elems / 8;
  P.per = ceil_div(P.b_vecs, (few ? 1024 : 256) * kScanVecs);
  P.seg = seg;
  P.bad = bad;
  P.ny = ceil_div(r8, kRankTile);
  P.nz = few ? std::min(N, int64_t(16)) : 1;
  const int64_t blocks = P.n_tiles * P.ny * P.nz + N * P.per;
  MIRL_REQUIRE(blocks < (few ? kMaxBlocks / 4 : kMaxBlocks), "too many rows or adapters");
  const dim3 grid((unsigned)blocks);
  with_rank(dtype, r8, [&](auto e, auto nt) {
    using E = decltype(e);
    constexpr int NT = decltype(nt)::value;
    if (few)
      hipLaunchKernelGGL((adapter_down_kernel<E, NT, 16>), grid, dim3(1024), 0, static_cast<hipStream_t>(stream), P);
    else
      hipLaunchKernelGGL((adapter_down_kernel<E, NT, 4>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), P);
  });
  return check_launch("mirl_adapter_down");
}

extern "C" int mirl_adapter_ce_fwd(const void* hidden, int dtype, int64_t T, int64_t Hd, int64_t ldh, const void* weight,
                                   int64_t V, int64_t ldw, const int32_t* adapter, const void* u_planes, const void* b,
                                   int64_t r8, int64_t N, const int32_t* bad, const int64_t* perm, const int64_t* target_rows, int64_t bsz,
                                   const int64_t* target, int64_t t_stride_b, int64_t t_stride_s, int64_t vocab_start,
                                   int64_t vocab_end, float* out, int64_t o_stride_b, int64_t o_stride_s,
                                   float* row_stats, float* workspace, void* stream) {
  clear_error();
  if (int e = check_operands(dtype, hidden, Hd, ldh, weight, V, ldw)) return e;
  MIRL_REQUIRE(T > 0 && T < kMaxRows && bsz > 0 && r8 > 0 && r8 % 8 == 0 && r8 <= kMaxRank,
               "invalid shape T=%lld B=%lld r8=%lld", (long long)T, (long long)bsz, (long long)r8);
  MIRL_REQUIRE(N > 0 && hidden && weight && adapter && u_planes && b && bad && perm && target_rows && target && out && workspace,
               "null pointer argument");
  MIRL_REQUIRE(aligned16(u_planes) && aligned16(b), "the adapters must be 16-byte aligned");
  LceParams P{};
  P.h = hidden;
  P.w = weight;
  P.ldh = ldh;
  P.ldw = ldw;
  P.V = V;
  P.Hd = padded_hidden(Hd, 2);
  P.Hw = Hd;
  P.nrows = T;
  P.bsz = 1;
  P.target = target_rows;
  P.tss = 1;
  P.vs = vocab_start;
  P.ve = vocab_end;
  P.aid = adapter;
  P.U = static_cast<const uint16_t*>(u_planes);
  P.B = static_cast<const uint16_t*>(b);
  P.r8 = (int)r8;
  P.planes = kPlanes;
  P.bad = bad;
  P.b_bytes = N * V * r8 * 2;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t tiles = dtype == MIRL_DTYPE_BF16 ? launch_fwd_x<BF16>(P, workspace, st) : launch_fwd_x<F16>(P, workspace, st);
  MIRL_REQUIRE(tiles < (int64_t(1) << 24), "too many tiles");
  auto merge = [&](auto kernel, int64_t blocks) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, P.part, P.xt, (int64_t)0, T, P.n_nt, bsz, target,
                       t_stride_b, t_stride_s, vocab_start, vocab_end, V, out, o_stride_b, o_stride_s, row_stats, perm);
  };
  if (T <= kJoinRows)
    merge(lce_merge_kernel<4>, T);
  else
    merge(lce_merge_kernel<1>, ceil_div(T, 4));
  return check_launch("mirl_adapter_ce_fwd");
}

extern "C" int mirl_adapter_gather(const int64_t* perm, const int32_t* adapter, const int64_t* count, int64_t T,
                                   const void* hidden, int dtype, int64_t Hd, int64_t ldh, const float* u_rows,
                                   int64_t r8, void* hidden_out, int64_t ldo, void* u_planes, void* stream) {
  clear_error();
  MIRL_REQUIRE(is16(dtype), "hidden states must be bf16 or fp16 (dtype code %d)", dtype);
  MIRL_REQUIRE(T > 0 && Hd > 0 && ldh >= Hd && ldo >= Hd && ldo % 8 == 0 && r8 > 0, "invalid shape");
  MIRL_REQUIRE(perm && adapter && count && hidden && u_rows && hidden_out && u_planes, "null pointer argument");
  MIRL_REQUIRE(r8 % 8 == 0 && aligned16(hidden_out) && aligned16(u_planes), "the gathered rows must be 16-byte aligned");
  auto launch = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL(adapter_gather_kernel<E>, dim3((unsigned)std::min(T, int64_t(1) << 20)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), perm, adapter, count, static_cast<const uint16_t*>(hidden), Hd,
                       ldh, u_rows, r8, static_cast<uint16_t*>(hidden_out), ldo, static_cast<uint16_t*>(u_planes));
  };
  if (dtype == MIRL_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return check_launch("mirl_adapter_gather");
}

extern "C" int mirl_transpose16(const void* src, int64_t Z, int64_t src_z, int64_t R, int64_t C, int64_t lds, void* dst,
                                int64_t dst_z, int64_t ldd, int64_t R_pad, const int64_t* count, const int64_t* perm,
                                double p, int64_t seed, const int64_t* seed_dev, int64_t offset, void* stream) {
  clear_error();
  MIRL_REQUIRE(Z >= 0 && R >= 0 && C >= 0 && R_pad >= R && lds >= C && ldd >= R_pad, "invalid shape");
  MIRL_REQUIRE(p >= 0.0 && p <= 1.0, "dropout probability %g is outside [0, 1]", p);
  if (Z == 0 || C == 0 || R_pad == 0) return MIRL_OK;
  MIRL_REQUIRE(src && dst, "null pointer argument");
  MIRL_REQUIRE(R_pad % 8 == 0 && ldd % 8 == 0 && dst_z % 8 == 0 && aligned16(dst),
               "transposed rows must be whole 16-byte pieces");
  TransposeParams P{static_cast<const uint16_t*>(src), R, C, lds, src_z, static_cast<uint16_t*>(dst), ldd, R_pad, dst_z,
                    ceil_div(C, 64), ceil_div(R_pad, 64), count, perm, dropout_args(p, seed, seed_dev, offset)};
  MIRL_REQUIRE(Z * P.n_ct * P.n_rt < kMaxBlocks, "too many tiles");
  hipLaunchKernelGGL(adapter_transpose_kernel, dim3((unsigned)(Z * P.n_ct * P.n_rt)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), P);
  return check_launch("mirl_transpose16");
}

extern "C" int mirl_adapter_ce_grad(const void* hidden, int dtype, int64_t Hd, int64_t ldh, const void* weight, int64_t V,
                                    int64_t ldw, const int32_t* adapter, const void* u_planes, const void* b, int64_t r8,
                                    int64_t N, const int32_t* bad, const int64_t* target_rows, int64_t vocab_start, int64_t vocab_end,
                                    const float* row_stats, int64_t row0, int64_t nrows, void* grad_logits, int64_t ldg,
                                    void* grad_logits_t, int64_t ldgt, const int64_t* row_count, void* stream) {
  clear_error();
  if (int e = check_operands(dtype, hidden, Hd, ldh, weight, V, ldw)) return e;
  MIRL_REQUIRE(row0 >= 0 && nrows > 0 && row0 + nrows < kMaxRows && r8 > 0 && r8 % 8 == 0 && r8 <= kMaxRank,
               "invalid shape row0=%lld rows=%lld r8=%lld", (long long)row0, (long long)nrows, (long long)r8);
  MIRL_REQUIRE(N > 0 && hidden && weight && adapter && u_planes && b && bad && target_rows && row_stats && grad_logits && grad_logits_t &&
                   row_count,
               "null pointer argument");
  MIRL_REQUIRE(ldg >= V, "gradient row stride %lld is smaller than V=%lld", (long long)ldg, (long long)V);
  MIRL_REQUIRE(ldgt >= round_up(nrows, kBM) && ldgt % 8 == 0 && aligned16(grad_logits_t),
               "transposed gradient: row stride %lld must cover %lld rows in whole 256-row tiles, be a multiple of 8 "
               "elements and start 16-byte aligned",
               (long long)ldgt, (long long)nrows);
  MIRL_REQUIRE(aligned16(u_planes) && aligned16(b), "the adapters must be 16-byte aligned");
  LceParams P{};
  P.h = hidden;
  P.w = weight;
  P.ldh = ldh;
  P.ldw = ldw;
  P.V = V;
  P.Hd = padded_hidden(Hd, 2);
  P.Hw = Hd;
  P.row0 = row0;
  P.nrows = nrows;
  P.bsz = 1;
  P.target = target_rows;
  P.tss = 1;
  P.vs = vocab_start;
  P.ve = vocab_end;
  P.n_mt = ceil_div(nrows, kBM);
  P.n_nt = ceil_div(V, kBN);
  P.stats = row_stats;
  P.G = static_cast<uint16_t*>(grad_logits);
  P.ldg = ldg;
  P.Gt = static_cast<uint16_t*>(grad_logits_t);
  P.ldgt = ldgt;
  P.count = row_count;
  P.aid = adapter;
  P.U = static_cast<const uint16_t*>(u_planes);
  P.B = static_cast<const uint16_t*>(b);
  P.r8 = (int)r8;
  P.planes = kPlanes;
  P.bad = bad;
  P.b_bytes = N * V * r8 * 2;
  const int64_t grid = ceil_div(P.n_mt * P.n_nt, kXcds) * kXcds;
  MIRL_REQUIRE(grid < (int64_t(1) << 24), "too many tiles");
  auto launch = [&](auto e) {
    using E = decltype(e);
    P.g_scale = g_scale_of<E>();
    const auto kernel = P.Hw != P.Hd ? lce_tile_kernel<kGradX, E, true> : lce_tile_kernel<kGradX, E, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream), P);
  };
  if (dtype == MIRL_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return check_launch("mirl_adapter_ce_grad");
}

extern "C" int mirl_gemm_f16_abt(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K,
                                 int64_t k_splits, float* C, int64_t ldc, const int64_t* count, int64_t count_off,
                                 void* stream) {
  clear_error();
  MIRL_REQUIRE(M >= 0 && N >= 0 && K > 0 && k_splits >= 1, "invalid shape M=%lld N=%lld K=%lld splits=%lld", (long long)M,
               (long long)N, (long long)K, (long long)k_splits);
  if (M == 0 || N == 0) return MIRL_OK;
  MIRL_REQUIRE(A && B && C, "null pointer argument");
  const int64_t kstep = (int64_t)kStages * kSK;
  MIRL_REQUIRE(K % kstep == 0, "reduction length %lld must be a multiple of %lld", (long long)K, (long long)kstep);
  const int64_t kb = round_up(ceil_div(K, k_splits), kstep), n_ks = ceil_div(K, kb);
  MIRL_REQUIRE(n_ks == k_splits, "%lld splits of K=%lld in ranges of %lld leave %lld non-empty", (long long)k_splits,
               (long long)K, (long long)kb, (long long)n_ks);
  MIRL_REQUIRE(lda % 8 == 0 && ldb % 8 == 0 && lda >= K && ldb >= K && ldc >= N,
               "row strides (%lld, %lld) must be multiples of 8 elements and >= K, the output's >= N", (long long)lda,
               (long long)ldb);
  MIRL_REQUIRE(aligned16(A) && aligned16(B), "operands must be 16-byte aligned");
  // buffer ranges of one 256-row tile are 32-bit byte counts
  MIRL_REQUIRE(kBM * lda * 2 < (int64_t(1) << 31) && kBN * ldb * 2 < (int64_t(1) << 31) && M < (int64_t(1) << 31) &&
                   N < (int64_t(1) << 31),
               "row strides (%lld, %lld) or sizes too large", (long long)lda, (long long)ldb);
  LceParams P{};
  P.h = A;
  P.w = B;
  P.ldh = lda;
  P.ldw = ldb;
  P.V = N;
  P.Hd = K;
  P.nrows = M;
  P.n_mt = ceil_div(M, kBM);
  P.n_nt = ceil_div(N, kBN);
  P.n_ks = n_ks;
  P.kb_len = kb;
  P.C = C;
  P.ldc = ldc;
  P.count = count;
  P.count_off = count_off;
  const int64_t grid = ceil_div(P.n_mt * P.n_nt * n_ks, kXcds) * kXcds;
  MIRL_REQUIRE(grid < (int64_t(1) << 24), "too many tiles");
  hipLaunchKernelGGL((lce_tile_kernel<kGemm, F16>), dim3((unsigned)grid), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), P);
  return check_launch("mirl_gemm_f16_abt");
}

// The block scratch: dU's partial sums and dU, the two transposed plane arrays, the maxima.
static int64_t block_floats(int64_t n, int64_t r8, int64_t splits) { return (splits + 1) * n * r8; }
static int64_t block_halves(int64_t n, int64_t r8) { return 2 * kPlanes * padded_rank(r8) * (round_up(n, 64) + 64); }

extern "C" int64_t mirl_adapter_block_workspace_bytes(int64_t n, int64_t r8, int64_t splits) {
  if (n <= 0 || r8 <= 0 || splits <= 0) return 0;
  return round_up(block_floats(n, r8, splits) * 4, 256) + round_up(block_halves(n, r8) * 2, 256) + n * 8;
}

extern "C" int mirl_adapter_block_grads(int dtype, int64_t row0, int64_t n, const int64_t* count, const int64_t* perm,
                                        const int32_t* adapter, const int32_t* seg, int64_t N, int64_t V, int64_t Hd,
                                        int64_t r, int64_t r8, const float* grad_rows, const float* scaling,
                                        const void* grad_logits, int64_t ldg, const void* grad_logits_t, int64_t ldgt,
                                        const void* b_t, int64_t ldbt, const void* a, int64_t lda, const void* hidden_t, int64_t ldht,
                                        const float* u_rows, double p, int64_t seed, const int64_t* seed_dev,
                                        int64_t offset, int64_t splits, const float* h_part, int64_t h_splits, void* dh,
                                        int64_t lddh, float* da, float* db, void* workspace, void* stream) {
  clear_error();
  MIRL_REQUIRE(is16(dtype), "hidden states must be bf16 or fp16 (dtype code %d)", dtype);
  MIRL_REQUIRE(row0 >= 0 && n > 0 && n < kMaxRows && N > 0 && V > 0 && Hd > 0 && r > 0 && r8 >= r && r8 % 8 == 0 && splits > 0,
               "invalid shape row0=%lld n=%lld N=%lld V=%lld H=%lld r=%lld", (long long)row0, (long long)n, (long long)N,
               (long long)V, (long long)Hd, (long long)r);
  MIRL_REQUIRE(r8 <= kMaxRank && lda >= Hd, "rank %lld (at most %lld) or row stride %lld", (long long)r,
               (long long)kMaxRank, (long long)lda);
  MIRL_REQUIRE(p >= 0.0 && p <= 1.0, "dropout probability %g is outside [0, 1]", p);
  MIRL_REQUIRE(count && perm && adapter && seg && grad_rows && scaling && grad_logits && b_t && a && u_rows && workspace &&
                   (db == nullptr || grad_logits_t) && (da == nullptr || hidden_t) && (dh == nullptr || h_part),
               "null pointer argument");
  MIRL_REQUIRE(ldbt % 128 == 0 && ldg >= ldbt && ldbt >= V && ldg % 8 == 0 && aligned16(grad_logits) && aligned16(b_t) &&
                   (db == nullptr || (ldgt >= round_up(n, 64) && ldgt % 8 == 0 && aligned16(grad_logits_t))) &&
                   (da == nullptr || (ldht >= row0 + round_up(n, 64) && ldht % 8 == 0 && row0 % 8 == 0 && aligned16(hidden_t))),
               "operand rows must be whole 16-byte pieces that cover the padded block");
  MIRL_REQUIRE(dh == nullptr || (lddh >= Hd && aligned16(h_part) && (Hd % 8 != 0 || (lddh % 8 == 0 && aligned16(dh)))),
               "invalid dH layout");
  BlockParams P{};
  P.row0 = row0;
  P.n = n;
  P.count = count;
  P.perm = perm;
  P.aid = adapter;
  P.seg = seg;
  P.N = N;
  P.V = V;
  P.H = Hd;
  P.r = r;
  P.r8 = r8;
  P.g = grad_rows;
  P.scaling = scaling;
  P.G = static_cast<const uint16_t*>(grad_logits);
  P.ldg = ldg;
  P.Gt = static_cast<const uint16_t*>(grad_logits_t);
  P.ldgt = ldgt;
  P.BT = static_cast<const uint16_t*>(b_t);
  P.ldbt = ldbt;
  P.A = static_cast<const uint16_t*>(a);
  P.lda = lda;
  P.hT = static_cast<const uint16_t*>(hidden_t);
  P.ldht = ldht;
  P.U32 = u_rows;
  P.drop = dropout_args(p, seed, seed_dev, offset);
  P.splits = splits;
  P.k_len = round_up(ceil_div(ldbt, splits), 128);
  P.du_part = static_cast<float*>(workspace);
  P.du = P.du_part + splits * n * r8;
  P.duT = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + round_up(block_floats(n, r8, splits) * 4, 256));
  P.r16 = padded_rank(r8);
  P.ldn = round_up(n, 64) + 64;
  P.ugT = P.duT + kPlanes * P.r16 * P.ldn;
  P.peak = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(P.duT) + round_up(block_halves(n, r8) * 2, 256));
  P.h_part = h_part;
  P.h_splits = h_splits;
  P.dH = dh;
  P.lddh = lddh;
  P.dA = da;
  P.dB = db;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned ny = (unsigned)ceil_div(r8, kRankTile);
  // dB: about four workgroups a CU (774 rows of 3 adapters, V = 32003: 31 -> 21 us)
  const unsigned nz = (unsigned)std::min(N, std::max(int64_t(1), 1024 / (ceil_div(V, 128) * ny)));
  // dH: four rows a workgroup read A once for them; one, where that leaves CUs idle (774 rows of
  // H = 1000 with 16 splits: 24.6 -> 17.7 us)
  const int64_t n_ct = ceil_div(Hd, 2048);
  const bool few = ceil_div(n, kDhRows) * n_ct < 1024;
  MIRL_REQUIRE(ceil_div(n, 128) * splits * ny < kMaxBlocks && ceil_div(V, 128) * ny < kMaxBlocks &&
                   ceil_div(Hd, 16) * ny < kMaxBlocks / 4 && ceil_div(n, kDhRows) * n_ct < kMaxBlocks,
               "too many tiles");
  with_rank(dtype, r8, [&](auto e, auto nt_c) {
    using E = decltype(e);
    constexpr int NT = decltype(nt_c)::value;
    const dim3 flat((unsigned)std::min(ceil_div(n * P.r16, 256), int64_t(4096)));
    hipLaunchKernelGGL((adapter_du_kernel<E, NT>), dim3((unsigned)(ceil_div(n, 128) * splits), ny), dim3(256), 0, st, P);
    hipLaunchKernelGGL(adapter_du_sum_kernel<E>, flat, dim3(256), 0, st, P);
    if (da != nullptr || db != nullptr) hipLaunchKernelGGL(adapter_planes_kernel<E>, flat, dim3(256), 0, st, P);
    if (db != nullptr)
      hipLaunchKernelGGL((adapter_db_kernel<E, NT>), dim3((unsigned)ceil_div(V, 128), ny, nz), dim3(256), 0, st, P);
    if (da != nullptr)
      hipLaunchKernelGGL((adapter_da_kernel<E, NT>), dim3((unsigned)ceil_div(Hd, 16), ny), dim3(kDaWaves * 64), 0, st, P);
    if (dh != nullptr && few)
      hipLaunchKernelGGL((adapter_dh_kernel<E, 1>), dim3((unsigned)(n * n_ct)), dim3(256), (unsigned)(r8 * 4), st, P);
    else if (dh != nullptr)
      hipLaunchKernelGGL((adapter_dh_kernel<E, kDhRows>), dim3((unsigned)(ceil_div(n, kDhRows) * n_ct)), dim3(256),
                         (unsigned)(kDhRows * r8 * 4), st, P);
  });
  return check_launch("mirl_adapter_block_grads");
}
