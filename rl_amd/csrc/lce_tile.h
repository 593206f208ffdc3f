// The MFMA tile loop of the hidden-state paths: a 256 x 256 tile of A . B^T and what becomes
// of it (see linear_ce.hip for the mathematics of each mode).
#pragma once

#include <algorithm>
#include <type_traits>
#include <utility>

#include "common.h"

#pragma clang fp contract(off)

namespace mirl {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Operand dtype of the tile loop: its fragment (16 bytes of a row per lane), the
// MFMA tile of kT x kT outputs and its accumulator.  run(w, h, c) forms
// c += W . H^T, W's rows along the accumulator's first index.
//
// 16-bit operands: v_mfma_f32_16x16x32.  Lane l holds elements k = (l / 16) * 8 + 0..7
// of row l % 16 of either operand, and accumulator element v of lane l is
// [W row (l / 16) * 4 + v][H row l % 16]: four consecutive vocabulary columns of one
// logits row.  (v_mfma_f32_32x32x16 does the same work per cycle with half the
// instructions, but the chip runs slower under it: forward of [16384, 4096] x
// [151808, 4096] 15.3 ms against 14.6 with the same epilogue.  Four columns per lane
// make the epilogue's LDS writes 8-byte pieces and its row data one set per eight
// tiles, and the plain GEMM's stores 8- or 16-byte pieces: forward 14.0 ms, 1450
// TFLOP/s; gradient 6.85 -> 6.1 ms of 5888 rows; dW 6.4 -> 5.65; dH 6.1 -> 5.65.)
template <class E>
struct Mma;
template <>
struct Mma<BF16> {
  typedef __bf16 frag __attribute__((ext_vector_type(8)));
  typedef f32x4 acc_t;
  static constexpr int kT = 16;
  __device__ __forceinline__ static f32x4 run(frag w, frag h, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, h, c, 0, 0, 0);
  }
};
template <>
struct Mma<F16> {
  typedef _Float16 frag __attribute__((ext_vector_type(8)));
  typedef f32x4 acc_t;
  static constexpr int kT = 16;
  __device__ __forceinline__ static f32x4 run(frag w, frag h, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(w, h, c, 0, 0, 0);
  }
};
// fp32 operands (plain GEMM only): the planes of a tile go through 32 x 32 outputs
// (see the kernel), and so do the tiles that the planes do not cover: a 16-byte
// fragment holds four hidden elements of a row, k = (l / 32) * 4 + 0..3, and feeds
// four v_mfma_f32_32x32x2_f32, element e of both fragments to the e-th one.  That
// instruction takes A[l % 32][l / 32] and B[l / 32][l % 32] from lane l, so the
// four together sum the products over the fragment's eight hidden elements
// (element e of the lanes below 32 is k = e, of the others k = 4 + e).
// Accumulator element v of lane l is
// [W row (v / 4) * 8 + (l / 32) * 4 + v % 4][H row l % 32].
template <>
struct Mma<F32> {
  typedef float frag __attribute__((ext_vector_type(4)));
  typedef f32x16 acc_t;
  static constexpr int kT = 32;
  __device__ __forceinline__ static f32x16 run(frag w, frag h, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(w[0], h[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(w[1], h[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(w[2], h[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(w[3], h[3], c, 0, 0, 0);
    return c;
  }
};
// e4m3 operands (OCP, forward of the 8-bit path only): v_mfma_f32_32x32x64_f8f6f4, unscaled,
// twice the bf16 rate.  A fragment is 32 bytes of a row per lane (two neighbouring 16-byte
// chunks); which hidden elements a lane holds does not matter as long as both operands hold
// the same ones.  The accumulator is laid out as for fp32.
struct F8 {
  using raw = uint8_t;
};
template <>
struct Mma<F8> {
  typedef int frag __attribute__((ext_vector_type(8)));
  typedef f32x16 acc_t;
  static constexpr int kT = 32;
  __device__ __forceinline__ static f32x16 run(frag w, frag h, f32x16 c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, h, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
  }
};

// Whether a partial pair (maximum, sum of exponentials) has a share in its row: all columns of one
// without are absent or -inf (a sum of 0).  A group of NaN has a maximum of -inf too, and NaN as its sum.
__device__ __forceinline__ bool counts(float m, float s) { return m != -INFINITY || s != 0.f; }

// 16-bit element bits <-> fp32 for a dtype E (round to nearest even).
template <class E>
__device__ __forceinline__ uint16_t bits_of(float f) {
  return __builtin_bit_cast(uint16_t, E::from_float(f));
}
template <class E>
__device__ __forceinline__ float value_of(uint16_t b) {
  return E::load_raw(__builtin_bit_cast(typename E::raw, b));
}
// Four fp32 values rounded to E, packed.
template <class E>
__device__ __forceinline__ uint2 pack4(f32x4 o) {
  if constexpr (std::is_same<E, BF16>::value)
    return uint2{BF16::pack2(o[0], o[1]), BF16::pack2(o[2], o[3])};
  else
    return uint2{(uint32_t)bits_of<E>(o[0]) | ((uint32_t)bits_of<E>(o[1]) << 16),
                 (uint32_t)bits_of<E>(o[2]) | ((uint32_t)bits_of<E>(o[3]) << 16)};
}
constexpr uint32_t kF16Past = 0x477ff000u;  // 65520, which fp16 rounds to infinity (bits of the fp32 value)
// A row of U past fp16's range (r8 values) enters the reduction times this power of two, which takes its
// largest finite magnitude to [2^14, 2^15); rows within the range times 1.
__device__ __forceinline__ float wide_scale(const float* u, int r8) {
  uint32_t peak = 0;
  for (int i = 0; i < r8; i += 4) {
    const float4 q = *reinterpret_cast<const float4*>(u + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t b = __float_as_uint(e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w) & 0x7fffffffu;
      peak = b < 0x7f800000u && b > peak ? b : peak;
    }
  }
  return peak < kF16Past ? 1.f : __uint_as_float((14 + 2 * 127 - (peak >> 23)) << 23);
}
// Eight values of u times `scale`: plane 0 of the two that add up to them, or plane 1.
template <class E>
__device__ __forceinline__ vu4 plane8(const float* u, float scale, int plane) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = u[i] * scale;
    const float first = value_of<E>(bits_of<E>(v[i]));
    v[i] = plane == 0 ? first : v[i] - first;
  }
  return E::pack(v);
}
typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr int kBM = 256;                 // rows per tile
constexpr int kBN = 256;                 // vocabulary columns per tile
constexpr int kSK = 64;                  // 16-bit hidden elements per LDS stage (128 bytes)
constexpr int kStages = 2;
constexpr int kThreads = 256;            // 4 waves in a 2 x 2 arrangement
constexpr int kWaves = kThreads / kWave;
constexpr int kWM = 128, kWN = 128;      // per-wave quarter
constexpr int kRowBytes = kSK * 2;       // 128 B: one tile row of a stage
constexpr int kHalfBytes = kBM * kRowBytes;    // 32 KB: the H (or W) rows of a stage
constexpr int kStageBytes = 2 * kHalfBytes;    // 64 KB
constexpr int kDmaBytes = kWave * 16;          // one direct load: 64 lanes x 16 B = 8 rows
constexpr int kDmaRows = kDmaBytes / kRowBytes;
constexpr int kDmaPerWave = kHalfBytes / kDmaBytes / kWaves;  // loads of H (and of W) per wave and stage
constexpr int kEpiRows = kStageBytes / (kBN * 2);  // epilogue tile rows held by one stage array
constexpr int kGroupM = 8;               // row tiles sharing a sweep over the vocabulary
constexpr int kXcds = 8;                 // accelerator dies, each with its own L2
static_assert(kBM == kBN, "H and W halves of a stage have the same size");
static_assert(kEpiRows * kStages == kBM, "the epilogue tile fills the stage arrays");
static_assert(kEpiRows == kWM, "a wave's epilogue rows live in one stage array");

// LDS byte offset (within a stage half) of 16-byte chunk `chunk` of tile row
// `row`.  A ds_read_b128 serves 16 lanes per pass (16 x 16 B = the 64
// four-byte banks); an MFMA operand read has those lanes on 16 consecutive rows
// at one chunk.  Two 128-byte rows span the 64 banks, so the chunk is XOR-ed
// with (row / 2) % 8: the 8 even and the 8 odd rows then each hit 8 distinct
// chunks, i.e. 16 distinct bank groups.
__device__ __forceinline__ int lds_off(int row, int chunk) {
  return row * kRowBytes + ((chunk ^ ((row >> 1) & 7)) << 4);
}

// Epilogue layout of the [256][256] bf16 tile: row r lives in stage array
// r / 128 at local row r % 128, row-major, 16-byte chunks XOR-swizzled by xs_swizzle(r)
// (element index within the array).  16 consecutive rows at one chunk (the
// accumulators' writes, the forward's row walk) and 8 rows 8 apart at two chunks (the
// transposed read) each fall in distinct banks.
__device__ __forceinline__ int xs_swizzle(int row) { return (row ^ (row >> 3)) & 31; }
__device__ __forceinline__ int xs_index(int row, int col) {
  return (row & (kEpiRows - 1)) * kBN + ((((col >> 3) ^ xs_swizzle(row)) << 3) | (col & 7));
}

// s_waitcnt vmcnt(N) lgkmcnt(0), then s_barrier.  The memory clobber keeps the
// compiler from moving LDS accesses across the barrier.
template <int N>
__device__ __forceinline__ void wait_vm_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The low bf16 of a pair, widened.  By a byte permute: for a shift, the compiler would
// form the low half once more with a conversion of its own.
__device__ __forceinline__ float low_bf16(uint32_t w) {
  return __uint_as_float(__builtin_amdgcn_perm(0u, w, 0x01000c0cu));
}

// w | the bits of a and b.  In asm: the compiler would gather the values to join first,
// on the stack.
__device__ __forceinline__ uint32_t or3(uint32_t w, float a, float b) {
  asm("v_or3_b32 %0, %0, %1, %2" : "+v"(w) : "v"(a), "v"(b));
  return w;
}

// A value that every lane of the wave holds, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>): a loop whose index
// the body may use in a constant expression.
template <int... I, class F>
__device__ __forceinline__ void static_for_(std::integer_sequence<int, I...>, F&& f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_(std::make_integer_sequence<int, N>{}, f);
}

// Flags of an adapter: its B holds an infinity or a NaN; fp16: a row's U is finite and past fp16's range.
constexpr int kBroken = 1, kWide = 2;
constexpr int kPlanes = 2;
// 16-bit rows of r8 that a row of U takes: its planes, and for fp16 its fp32 values (u_f32).
template <class E>
constexpr int kURow = std::is_same<E, F16>::value ? 4 : 2;
template <class T>
__device__ __forceinline__ auto u_f32(T* U, int64_t row, int r8) {
  using F = typename std::conditional<std::is_const<T>::value, const float, float>::type;
  return reinterpret_cast<F*>(U + (row * kURow<F16> + kPlanes) * r8);
}

// kFwd, kGrad: logits rounded to the operand type.  kFwdX, kGradX: logits kept in fp32, with
// adapters (16-bit operands) or row and column scales (e4m3, forward).
enum LceMode { kFwd = 0, kGrad = 1, kGemm = 2, kFwdX = 3, kGradX = 4 };

struct LceParams {
  const void* h;  // [T, Hd] of the kernel's E (bf16, fp16; fp32 for the plain GEMM), row stride ldh
  const void* w;  // [V, Hd] of the same dtype, row stride ldw
  int64_t ldh, ldw;
  int64_t V, Hd;
  int64_t row0, nrows;  // rows handled: [row0, row0 + nrows)
  int64_t bsz;          // row r is (s, b) = (r / bsz, r % bsz)
  const int64_t* target;
  int64_t tsb, tss;
  int64_t vs, ve;
  int64_t n_mt, n_nt;   // row tiles, column tiles
  // forward
  float* part;          // [nrows, n_nt, 2]
  float* xt;            // [nrows]
  // gradient
  const float* stats;   // [T, 2] {max, logsum} by absolute row
  const float* g;
  int64_t gsb, gss;
  uint16_t* G;          // [nrows, V] bf16, row stride ldg
  int64_t ldg;
  uint16_t* Gt;         // or null: G transposed, [V, ldgt] bf16 (column r - row0 of row v)
  int64_t ldgt;
  // plain GEMM (kGemm): C = A . B^T with A = h [nrows, Hd], B = w [V, Hd]; the
  // hidden dimension is split into n_ks ranges of kb_len (C holds n_ks
  // partial products [n_ks][nrows][ldc]), or Cb receives bf16(C) (n_ks = 1)
  int64_t n_ks, kb_len;
  float* C;
  uint16_t* Cb;        // bf16 output, fp16 with cb_f16
  int cb_f16;
  int64_t ldc, ldcb;
  int accumulate;       // C += A . B^T instead of C = A . B^T (n_ks = 1)
  // device count (or null): c = *count - count_off.  kFwd/kGrad and count_axis
  // 0: rows r >= c are absent (not read, not written); count_axis 1 (kGemm):
  // the reduction stops at round_up(c, 128).  With both C and Cb, the output
  // is Cb = bf16(A . B^T (+ C when accumulate)) if *count <= final_at and C
  // otherwise; an empty reduction with accumulate set writes nothing.
  const int64_t* count;
  int64_t count_off;
  int count_axis;
  int64_t final_at;
  // kFwdX and kGradX with adapters (or null): row r takes adapter aid[r] (rows of one
  // adapter adjoin; negative: none), which adds U[r] . B[aid[r]]^T to its logits.  U is held as
  // `planes` values of the operand type that add up to it: row r is [kURow<E>][r8], the planes
  // first (fp16: then U in fp32); B is [adapters, V, r8], r8 a multiple of 8.
  const int32_t* aid;
  const uint16_t* U;
  const uint16_t* B;
  int r8, planes;
  const int32_t* bad;   // [adapters]: kBroken, kWide
  int64_t b_bytes;      // size of B
  // kGradX: G = (onehot - softmax) * g_scale in the operand type (rows past the end: 0)
  float g_scale;
  // kFwdX and kGradX: W's rows hold Hw elements (whole 16-byte chunks), H's Hd, zeros past Hw
  int64_t Hw;
  // kFwdX of e4m3: logits = products * col_scale[col] * row_scale[row]
  const float* row_scale;
  const float* col_scale;
};

// RAGGED (kFwdX, kGradX): Hw is not a whole number of stage pairs.  What lies past a row of W is then
// masked in the last two stages' loads: it is the next row's beginning, or no part of W, and an
// infinity or a NaN there must not meet the zeros of H's rows.
template <int MODE, class E, bool RAGGED = false>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1, 1)))
void lce_tile_kernel(LceParams P) {
  using frag = typename Mma<E>::frag;
  using acc_t = typename Mma<E>::acc_t;
  constexpr int kT = Mma<E>::kT, kTM = kWM / kT, kTN = kWN / kT, kAV = kT * kT / kWave;
  constexpr int kKK = kRowBytes / (kWave / kT * (int)sizeof(frag));  // fragment steps (MFMA blocks) per stage
  constexpr int kES = (int)sizeof(typename E::raw);  // bytes per element
  static_assert(MODE == kGemm ? kES != 1 : MODE == kFwdX ? kES <= 2 : kES == 2,
                "fp32 operands: plain GEMM only; e4m3: forward only");
  constexpr bool kIsGrad = MODE == kGrad || MODE == kGradX;
  constexpr bool kAdapters = (MODE == kFwdX || MODE == kGradX) && kES == 2;
  constexpr int kSKE = kRowBytes / kES;              // hidden elements per stage
  // Two arrays rather than one, so that the compiler tracks the direct loads
  // into each stage on their own and an LDS read waits only for its stage.
  __shared__ __align__(1024) unsigned char st0[kStageBytes];
  __shared__ __align__(1024) unsigned char st1[kStageBytes];
  __shared__ int s_tcol[kBM];
  __shared__ __align__(16) float s_m[kBM], s_ls[kBM], s_g[kBM], s_rs[MODE == kFwdX && kES == 1 ? kBM : 1];
  __shared__ int s_ord[kAdapters ? kBM : 1], s_seg[kAdapters ? kBM : 1], s_bad[kAdapters ? kBM : 1],
      s_heads[kWaves];
  constexpr bool kF16 = kAdapters && std::is_same<E, F16>::value;
  const int ur = kF16 ? kURow<F16> : P.planes;
  __shared__ float s_us[kF16 ? kBM : 1];
  auto stage_ptr = [&](int s) -> unsigned char* { return s == 0 ? st0 : st1; };

  // Tile order.  Workgroups are dispatched to the 8 XCDs round-robin
  // (XCD = blockIdx % 8) and each XCD has its own L2, so each XCD takes one
  // contiguous run of a grouped order (kGroupM row tiles sweep the vocabulary
  // together): the ~32 workgroups resident on an XCD then cover about
  // kGroupM row tiles x 4 column tiles and share their H and W reads in L2.
  // (A plain GEMM's hidden-dimension splits are the outermost index.)
  // A device count of rows shortens the row range; the tile order then covers
  // only the row tiles that hold rows (so every XCD keeps its share of the
  // work) and the workgroups past them return at once.
  int64_t row_end = P.row0 + P.nrows;
  int64_t k_end = P.Hd;
  bool to_bf16 = P.Cb != nullptr;
  if (P.count != nullptr) {
    const int64_t c = *P.count - P.count_off;
    if (MODE != kGemm || P.count_axis == 0) {
      if (c < row_end) row_end = c;
    } else {
      constexpr int64_t kstep = kStages * kSKE;
      const int64_t ke = c <= 0 ? 0 : (c + kstep - 1) / kstep * kstep;
      if (ke < k_end) k_end = ke;
      if (ke == 0 && P.accumulate) return;
      if (P.C != nullptr && P.Cb != nullptr) to_bf16 = *P.count <= P.final_at;
    }
  }
  row_end = uniform(row_end);
  k_end = uniform(k_end);
  if (row_end <= P.row0) return;
  const int64_t n_mt = (row_end - P.row0 + kBM - 1) / kBM;  // <= P.n_mt
  const int64_t tiles2 = n_mt * P.n_nt;
  const int64_t ntiles = tiles2 * (MODE == kGemm ? P.n_ks : 1);
  const int64_t per_xcd = (ntiles + kXcds - 1) / kXcds;
  // (the grid holds per_xcd workgroups per XCD only without a count)
  if ((int64_t)(blockIdx.x / kXcds) >= per_xcd) return;
  const int64_t gi0 = (int64_t)(blockIdx.x % kXcds) * per_xcd + blockIdx.x / kXcds;
  if (gi0 >= ntiles) return;
  const int64_t ks = uniform(gi0 / tiles2);
  const int64_t gi = gi0 - ks * tiles2;
  const int64_t per_group = (int64_t)kGroupM * P.n_nt;
  const int64_t group = gi / per_group;
  const int64_t first_m = group * kGroupM;
  const int64_t gsize = (n_mt - first_m < kGroupM) ? (n_mt - first_m) : kGroupM;
  const int64_t in_group = gi - group * per_group;
  // wave-uniform by construction; said so, or the compiler may keep the buffer
  // resources made from them in vector registers and loop over lanes at every load
  const int64_t mt = uniform(first_m + in_group % gsize);
  const int64_t nt = uniform(in_group / gsize);
  const int64_t m0 = P.row0 + mt * kBM;  // absolute first row
  const int64_t n0 = nt * kBN;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wm = wave >> 1, wn = wave & 1;

  // per-row metadata of the tile (kThreads == kBM: one row per thread)
  float my_g = 0.f;
  int n_seg = 0;
  bool apart = false;  // the adapters' part is formed by itself (adapter_stages)
  auto metadata = [&]() __attribute__((always_inline)) {
    const int64_t r = m0 + tid;
    int tc = -1;
    float lm = 0.f, ll = 0.f;
    if (r < row_end) {
      const int64_t s = r / P.bsz, b = r - s * P.bsz;
      const int64_t t = P.target[b * P.tsb + s * P.tss];
      const bool tmask = (t < P.vs) || (t >= P.ve) || (t - P.vs >= P.V);
      if (!tmask) {
        const int64_t c = t - P.vs - n0;
        if (c >= 0 && c < kBN) tc = (int)c;
      }
      if (kIsGrad) {
        my_g = MODE == kGradX ? P.g_scale : P.g[b * P.gsb + s * P.gss];
        lm = P.stats[2 * r];
        ll = P.stats[2 * r + 1];
      }
    }
    s_tcol[tid] = tc;
    if (kIsGrad) {
      s_g[tid] = my_g;
      s_m[tid] = lm;
      s_ls[tid] = ll;
    }
    if constexpr (MODE == kFwdX && kES == 1) {
      s_rs[tid] = r < row_end ? P.row_scale[r] : 0.f;
      s_ls[tid] = n0 + tid < P.V ? P.col_scale[n0 + tid] : 0.f;
    }
    // The tile's adapters in row order: s_seg[q] is the q-th one, s_ord[row] the row's (-1: none).
    if constexpr (kAdapters) {
      const int a = r < row_end ? P.aid[r] : -1;
      const int before = tid > 0 && r < row_end ? P.aid[r - 1] : -1;
      const bool head = a >= 0 && (tid == 0 || a != before);
      const uint64_t heads = __ballot(head);
      if (lane == 0) s_heads[wave] = (int)__popcll(heads);
      __syncthreads();
      int at = (int)__popcll(heads & (~0ull >> (63 - lane)));  // heads up to this row
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        at += w < wave ? s_heads[w] : 0;
        n_seg += s_heads[w];
      }
      s_ord[tid] = a >= 0 ? at - 1 : -1;
      const int bad = head ? P.bad[a] : 0;
      if (head) {
        s_seg[at - 1] = a;
        s_bad[at - 1] = bad;
      }
      // (32-bit offsets reach 2 GiB of B)
      apart = __syncthreads_or(bad) != 0 || P.b_bytes >= (int64_t(1) << 31);
      n_seg = __builtin_amdgcn_readfirstlane(n_seg);
    }
  };
  if constexpr (MODE != kGemm) metadata();
  if (MODE == kGrad) {
    // (onehot - p) * 0 == 0: a tile whose rows all have a zero upstream
    // gradient is written as zeros without the GEMM.
    if (!__syncthreads_or(my_g != 0.f)) {
      const int cvec = kBN / 8;
      for (int q = tid; q < kBM * cvec; q += kThreads) {
        const int rl = q / cvec, cv = q - rl * cvec;
        const int64_t r = m0 + rl;
        const int64_t c = n0 + cv * 8;
        if (r >= row_end || c >= P.V) continue;
        uint16_t* dst = P.G + (r - P.row0) * P.ldg + c;
        if (c + 8 <= P.V && ((reinterpret_cast<uintptr_t>(dst) & 15u) == 0)) {
          *reinterpret_cast<vu4*>(dst) = vu4{0u, 0u, 0u, 0u};
        } else {
          for (int e = 0; e < 8 && c + e < P.V; ++e) dst[e] = 0;
        }
      }
      if (P.Gt != nullptr && n0 + tid < P.V) {
        uint16_t* dt = P.Gt + (n0 + tid) * P.ldgt + (m0 - P.row0);
        for (int r8 = 0; r8 < kBM / 8; ++r8) *reinterpret_cast<vu4*>(dt + r8 * 8) = vu4{0u, 0u, 0u, 0u};
      }
      return;
    }
  }

  // ---- main loop: acc = H[m0 : m0+256] . W[n0 : n0+256]^T ----
  //
  // Direct loads go through buffer resources covering the tile's valid rows.
  // The row offset is in the VGPR offset, which the range check covers, so rows
  // past the end of H or W read as zero with no branch; the SGPR offset carries
  // only the stage's hidden offset, which stays inside a valid row.
  //
  // One direct load moves 8 rows x 128 B: lane l writes LDS bytes
  // [16 l, 16 l + 16) of the load's 1 KB block, i.e. row l / 8, slot l % 8, so
  // it fetches global chunk (l % 8) ^ ((row / 2) % 8) of that row (the inverse
  // of the lds_off swizzle).  Each wave issues kDmaPerWave loads of H and of W
  // per stage.
  // this tile's range of the hidden dimension (the whole of it but for split GEMMs)
  const int64_t kbase = (MODE == kGemm) ? ks * P.kb_len : 0;
  const int64_t krest = k_end - kbase < 0 ? 0 : k_end - kbase;
  const int64_t klen = (MODE == kGemm) ? (krest < P.kb_len ? krest : P.kb_len) : P.Hd;
  const int nst = (int)(klen / kSKE);  // a multiple of kStages (0: an empty reduction)
  if (MODE == kGemm && nst == 0) {
    // an empty reduction range (a reduction-length count, or a split past it):
    // the product is zero; handled here, before the accumulators exist
    for (int q = threadIdx.x; q < kBM * kBN; q += kThreads) {
      const int64_t row = m0 + q / kBN, col = n0 + q % kBN;
      if (row >= row_end || col >= P.V) continue;
      if (to_bf16) {
        const float o = (P.accumulate && P.C != nullptr) ? P.C[row * P.ldc + col] : 0.f;
        P.Cb[row * P.ldcb + col] = P.cb_f16 ? bits_of<F16>(o) : bits_of<BF16>(o);
      } else if (!P.accumulate) {
        P.C[(ks * P.nrows + row) * P.ldc + col] = 0.f;
      }
    }
    return;
  }
  const int64_t a_rows = (row_end - m0 < kBM) ? (row_end - m0) : kBM;
  const int64_t b_rows = (P.V - n0 < kBN) ? (P.V - n0) : kBN;
  __amdgpu_buffer_rsrc_t rsrc_a = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(P.h) + (m0 * P.ldh + kbase) * kES), 0,
      (int)((a_rows * P.ldh - kbase) * kES), 0x00020000);
  __amdgpu_buffer_rsrc_t rsrc_b = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(P.w) + (n0 * P.ldw + kbase) * kES), 0,
      (int)((b_rows * P.ldw - kbase) * kES), 0x00020000);
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  int voff_a[kDmaPerWave], voff_b[kDmaPerWave];
#pragma unroll
  for (int i = 0; i < kDmaPerWave; ++i) {
    const int row = (wave * kDmaPerWave + i) * kDmaRows + (lane >> 3);
    const int chunk = (lane & 7) ^ ((row >> 1) & 7);
    voff_a[i] = (int)(row * P.ldh * kES) + chunk * 16;
    voff_b[i] = (int)(row * P.ldw * kES) + chunk * 16;
  }
  constexpr int kOut = -0x7fffffff - 1;  // an offset out of range: reads as zero
  // RAGGED: from stage t on, one of the last two, the chunks past W's row are out of range.
  auto end_w = [&](int t) __attribute__((always_inline)) {
    int ln = lane;
    asm volatile("" : "+v"(ln));  // (see prepare)
    const int left = (int)(P.Hw * kES) - t * kRowBytes;
#pragma unroll
    for (int i = 0; i < kDmaPerWave; ++i) {
      // a load's rows start at a multiple of 8, so its chunks depend on its parity only
      const int chunk = (ln & 7) ^ (((ln >> 4) + 4 * (i & 1)) & 7);
      voff_b[i] = chunk * 16 >= left ? kOut : voff_b[i];
    }
  };
  // load q of stage data t: q < kDmaPerWave is an H block, else a W block
  auto dma = [&](unsigned char* stage, int t, int q) {
    const int soff = kAdapters && t >= nst ? 0 : t * kRowBytes;
    if (q < kDmaPerWave) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc_a, (lds_ptr_t)(stage + (wave_u * kDmaPerWave + q) * kDmaBytes), 16, voff_a[q], soff, 0, 0);
    } else {
      const int qb = q - kDmaPerWave;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc_b, (lds_ptr_t)(stage + kHalfBytes + (wave_u * kDmaPerWave + qb) * kDmaBytes), 16,
          voff_b[qb], soff, 0, 0);
    }
  };

  // Adapter stages: stage data nst + e continues the reduction over the tile's adapters one after
  // the other, `planes` * r8 elements each, eight 16-byte chunks a stage; a row's U is zero in the
  // chunks of other adapters (an offset out of range reads as zero).  One adapter of rank up to 16
  // takes half of one of the two stages added to 64 at a hidden size of 4096, several share them:
  // forward of [16384, 4096] x [151936, 4096] 14.3 ms against 14.0 without adapters.  (Formed
  // stage by stage ahead of the loop it took 15.7; with an odd number of stages allowed, the
  // accumulators no longer stay in place through the branches, 470 registers are spilled.)
  const int cpp = kAdapters ? P.r8 >> 3 : 1, cps = kAdapters ? P.planes * cpp : 1;
  const int n_ext = (n_seg * cps + 7) >> 3;
  const int total = kAdapters && !apart ? nst + (n_ext + 1) / 2 * 2 : nst;
  auto prepare = [&](int t) __attribute__((always_inline)) {
    // opaque here, or everything that follows from it is formed ahead of the main loop and
    // kept in registers that it lacks
    int ln = lane;
    asm volatile("" : "+v"(ln));
    rsrc_a = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(P.U + m0 * (int64_t)(ur * P.r8)), 0,
                                               (int)(a_rows * ur * P.r8 * 2), 0x00020000);
    rsrc_b = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(P.B + n0 * P.r8), 0,
                                               (int)(P.b_bytes - n0 * P.r8 * 2), 0x00020000);
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      // a load's rows start at a multiple of 8, so its chunks depend on its parity only
      const int x = (t - nst) * 8 + ((ln & 7) ^ (((ln >> 4) + 4 * odd) & 7));
      const int seg = x / cps, rem = x - seg * cps, cc = rem % cpp;
      const int b0 = (s_seg[seg < n_seg ? seg : 0] * (int)P.V * P.r8 + cc * 8) * 2;
#pragma unroll
      for (int i = odd; i < kDmaPerWave; i += 2) {
        const int row = (wave * kDmaPerWave + i) * kDmaRows + (ln >> 3);
        voff_a[i] = s_ord[row] == seg ? (row * ur * P.r8 + rem * 8) * 2 : kOut;
        voff_b[i] = ((seg < n_seg) & (row < (int)b_rows)) ? b0 + row * P.r8 * 2 : kOut;
      }
    }
  };

  // fragment read offsets: row (wm*128 | wn*128) + i*kT + lane % kT, the lane group's
  // chunk of step kk (e4m3: the first of two neighbouring chunks, the other at offset ^ 16)
  const int frow = lane & (kT - 1);
  constexpr int kFC = (int)sizeof(frag) / 16;  // chunks of a fragment
  int frag_off[kKK];
#pragma unroll
  for (int kk = 0; kk < kKK; ++kk) frag_off[kk] = lds_off(frow, (kk * (kWave / kT) + lane / kT) * kFC);
  frag fa[2][kTM], fb[2][kTN];
  // Reads go out in the order the MFMAs first need them: A0, all B, the other A (1% on
  // the forward against all A, all B).
  auto fread = [&](int set, const unsigned char* stage, int kk, int n) __attribute__((always_inline)) {
    // idx < kTM: A fragment idx; else B fragment idx - kTM
    const int idx = n == 0 ? 0 : n <= kTN ? kTM + n - 1 : n - kTN;
    const unsigned char* base = idx < kTM ? stage + (wm * kWM + idx * kT) * kRowBytes
                                          : stage + kHalfBytes + (wn * kWN + (idx - kTM) * kT) * kRowBytes;
    frag& f = idx < kTM ? fa[set][idx] : fb[set][idx - kTM];
    if constexpr (kFC == 1) {
      f = *reinterpret_cast<const frag*>(base + frag_off[kk]);
    } else {
      const vu4 a = *reinterpret_cast<const vu4*>(base + frag_off[kk]);
      const vu4 b = *reinterpret_cast<const vu4*>(base + (frag_off[kk] ^ 16));
      f = frag{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    }
  };

  acc_t acc[kTM][kTN];
  auto clear_acc = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
      for (int j = 0; j < kTN; ++j)
#pragma unroll
        for (int v = 0; v < kAV; ++v) acc[i][j][v] = 0.f;
  };
  clear_acc();
  auto mfma = [&](int set, int q) __attribute__((always_inline)) {
    const int i = q / kTN, j = q % kTN;
    acc[i][j] = Mma<E>::run(fb[set][j], fa[set][i], acc[i][j]);
  };

  constexpr int kL = 2 * kDmaPerWave;  // direct loads per wave and stage
  constexpr int kMB = kTM * kTN;        // MFMAs per block
  constexpr int kReadEvery = kMB / (2 * (kTM + kTN)) > 1 ? 2 : 1, kLoadEvery = kMB / kL;
  static_assert(kKK % 2 == 0 && kLoadEvery * kL == kMB && kReadEvery * (kTM + kTN) <= kMB,
                "a block's reads and loads fit beside its MFMAs");
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using T_ = std::integral_constant<bool, true>;
  using F_ = std::integral_constant<bool, false>;
  // One stage t (S = t % 2): kKK blocks of MFMAs (two of 64 for 16-bit operands, 32
  // hidden elements each).  While block kk runs on fragment set kk % 2, block kk + 1's
  // fragments are read into the other set.  Before the last block this wave waits for
  // its loads of stage data t + 1 (the only ones in flight) and the workgroup barrier
  // makes every wave's loads visible and ends every read of stage S (the last block's
  // fragments were read beside the block before).  The last block then reads the next
  // stage's block-0 fragments and issues the direct loads of stage data t + 2 into stage
  // S, spread over its MFMAs: 64 KB for the CU's LDS write port in half a stage.  (In a
  // quarter of the stage, forward 15.8 ms against 15.05, dW 6.42 against 5.88, dH 6.11
  // against 5.79 on [16384 | 5888, 4096] x [151808, 4096], all with 32 x 32 MFMAs; over
  // three quarters 15.57 ms: the last loads then come too late.)
  auto step = [&](int t, auto s_c, auto next_c, auto load_c) __attribute__((always_inline)) {
    constexpr int S = decltype(s_c)::value;
    constexpr bool NEXT = decltype(next_c)::value;
    constexpr bool LOAD = decltype(load_c)::value;
    unsigned char* cur = stage_ptr(S);
    const unsigned char* nxt = stage_ptr(S ^ 1);
#pragma unroll
    for (int kk = 0; kk < kKK - 1; ++kk) {
#pragma unroll
      for (int q = 0; q < kMB; ++q) {
        mfma(kk & 1, q);
        if (q % kReadEvery == 0 && q / kReadEvery < kTM + kTN) fread((kk + 1) & 1, cur, kk + 1, q / kReadEvery);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (NEXT) wait_vm_barrier<0>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < kMB; ++q) {
      mfma(1, q);
      if constexpr (NEXT) {
        if (q % kReadEvery == 0 && q / kReadEvery < kTM + kTN) fread(0, nxt, 0, q / kReadEvery);
      }
      if constexpr (LOAD) {
        if (q % kLoadEvery == kLoadEvery / 4) dma(cur, t + 2, q / kLoadEvery);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // The adapters' part by itself, stage by stage through stage array 1, where a value of an adapter
  // is none, B passes 2 GiB or (fp16) a row's U the type's range:
  // an infinity or a NaN of one adapter's B must not meet the other rows' zeros, so it is taken
  // out, and that adapter's rows become NaN afterwards (s_bad).  A row of U past the range comes from
  // fp32 times a power of two, and so does what the row has summed.
  auto nonfinite = [](vu4 q) __attribute__((always_inline)) {
    constexpr uint32_t ex = std::is_same<E, BF16>::value ? 0x7f80u : 0x7c00u;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
      bad |= (w & ex) == ex || ((w >> 16) & ex) == ex;
    }
    return bad;
  };
  // The accumulators are complete here, in the registers that the MFMAs write.
  auto keep_acc = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
      for (int j = 0; j < kTN; ++j) asm volatile("" : "+a"(acc[i][j]));
  };
  auto scale_rows = [&](bool back) __attribute__((always_inline)) {
    // One accumulator register at a time, by asm: left to itself the compiler moves all of them to other
    // registers around this branch and spills 130.  The waits stand between MFMAs and these accesses.
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
      float f = s_us[kF16 ? wm * kWM + i * kT + frow : 0];
      f = back ? 1.f / f : f;  // powers of two: exact
#pragma unroll
      for (int j = 0; j < kTN; ++j) {
#pragma unroll
        for (int v = 0; v < kAV; ++v) {
          float x;
          asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(acc[i][j][v]));
          x *= f;
          asm volatile("v_accvgpr_write_b32 %0, %1" : "=a"(acc[i][j][v]) : "v"(x));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_nop 15" ::: "memory");
  };
  auto adapter_stages = [&]() __attribute__((always_inline)) {
    const int chunk = tid & 7;
    bool wide = false;
    if constexpr (kF16) {
      const bool mine = s_ord[tid] >= 0 && (s_bad[s_ord[tid]] & kWide) != 0;
      s_us[tid] = mine ? wide_scale(u_f32(P.U, m0 + tid, P.r8), P.r8) : 1.f;
      wide = __syncthreads_or(mine) != 0;
      if (wide) scale_rows(false);
    }
    for (int e = 0; e < n_ext; ++e) {
      const int x = e * 8 + chunk, q = x / cps, rem = x - q * cps, cc = rem % cpp;
      const bool any = q < n_seg;
      const uint16_t* up = P.U + m0 * (int64_t)(ur * P.r8) + rem * 8;
      const uint16_t* bp = P.B + ((int64_t)(any ? s_seg[q] : 0) * P.V + n0) * P.r8 + cc * 8;
      __syncthreads();  // the last stage's reads are done
#pragma unroll 1
      for (int k = 0; k < kBM / 32; ++k) {
        const int row = k * 32 + (tid >> 3);
        vu4 u = {0u, 0u, 0u, 0u}, b = {0u, 0u, 0u, 0u};
        if (any && s_ord[row] == q) {
          u = *reinterpret_cast<const vu4*>(up + (int64_t)row * (ur * P.r8));
          if constexpr (kF16) {
            if (wide) u = plane8<E>(u_f32(P.U, m0 + row, P.r8) + cc * 8, s_us[row], rem / cpp);
          }
        }
        if (any && n0 + row < P.V) b = *reinterpret_cast<const vu4*>(bp + (int64_t)row * P.r8);
        if (nonfinite(b)) b = vu4{0u, 0u, 0u, 0u};
        *reinterpret_cast<vu4*>(st1 + lds_off(row, chunk)) = u;
        *reinterpret_cast<vu4*>(st1 + kHalfBytes + lds_off(row, chunk)) = b;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) {
#pragma unroll
        for (int n = 0; n < kTM + kTN; ++n) fread(0, st1, kk, n);
#pragma unroll
        for (int m = 0; m < kMB; ++m) mfma(0, m);
      }
    }
    __syncthreads();
    if constexpr (kF16) {
      if (wide) scale_rows(true);
    }
    if constexpr (MODE == kGradX) {
      if (s_ord[tid] >= 0 && (s_bad[s_ord[tid]] & kBroken) != 0) s_g[tid] = __builtin_nanf("");
    }
  };
  auto run_stages = [&]() __attribute__((always_inline)) {
    // Prologue: stage data 0 and 1 in flight; wait for 0 and read its block-0 fragments.
    if (RAGGED && nst == kStages) end_w(0);
#pragma unroll
    for (int q = 0; q < kL; ++q) dma(st0, 0, q);
    if (RAGGED && nst == kStages) end_w(1);
#pragma unroll
    for (int q = 0; q < kL; ++q) dma(st1, 1, q);
    wait_vm_barrier<kL>();
#pragma unroll
    for (int idx = 0; idx < kTM + kTN; ++idx) fread(0, st0, 0, idx);
    int t = 0;
    for (; t < nst - (RAGGED ? 2 : 1) * kStages; t += kStages) {
      step(t, S0{}, T_{}, T_{});
      step(t + 1, S1{}, T_{}, T_{});
    }
    if constexpr (RAGGED) {
      for (; t < nst - kStages; t += kStages) {  // the last two stages' loads
        end_w(t + kStages);
        step(t, S0{}, T_{}, T_{});
        end_w(t + 1 + kStages);
        step(t + 1, S1{}, T_{}, T_{});
      }
    }
    if constexpr (kAdapters) {
      for (; t < total - kStages; t += kStages) {
        prepare(t + kStages);
        step(t, S0{}, T_{}, T_{});
        prepare(t + 1 + kStages);
        step(t + 1, S1{}, T_{}, T_{});
      }
    }
    step(t, S0{}, T_{}, F_{});
    step(t + 1, S1{}, F_{}, F_{});
  };

  float unscale = 1.f;  // what the accumulators are to be multiplied by (fp32 operands)
  if constexpr (std::is_same<E, F32>::value) {
    // ---- fp32 operands as three bf16 planes each ----
    //
    // x = x0 + x1 + x2 exactly, with x0 = bf16(x), x1 = bf16(x - x0) and
    // x2 = x - x0 - x1 (at most eight significant bits are left), so a product of
    // two elements is the sum of nine bf16 products; the three below 2^-25 of it
    // (a1 b2, a2 b1, a2 b2) are left out and the six others summed into the same
    // fp32 accumulators, the small ones first.  The fp32 MFMA runs at 1/16 of the bf16
    // rate, so six bf16 products cost 3/8 of one fp32 product, and 32 k-terms enter an
    // accumulator in 12 roundings instead of 16: [2048, 4096] x [65536, 4096]^T 151 -> 241
    // TFLOP/s back to back (1450 of bf16), error against 64 bits 1.15e-6 -> 1.00e-6 of the root
    // of the sum of squared products (K = 64: 1.44e-7 -> 1.10e-7; sums of two terms 3.1e-8
    // -> 3.3e-8, of one 2.5e-8 -> 3.4e-8: what is left out counts there).  Bound by the MFMA
    // units, busy 87% of the cycles at the 1.5 GHz that this load leaves (82% at 1.92 GHz
    // and 276 TFLOP/s where memory-bound kernels run in between).
    //
    // Unscaled, the planes hold all of x from 2^-109 on, and the logits gradient (the
    // first operand of dH and dW) is less for every improbable token: one such value
    // sends its tile through both loops below.  So the first operand is multiplied by
    // 2^40 before it is split and the result by 2^-40: its planes then hold every x below
    // 2^88, subnormal ones too.  Step of [1024, 2, 4096] x [151936, 4096], every row
    // active: with logits of standard deviation 10 83.1 -> 50.5 ms, of 1.5 49.4 and 49.3.
    // (Both operands by 2^24, without the check of the residuals, takes 3% more.)
    //
    // Each lane reads the fp32 fragments of the coming 16 hidden elements and
    // splits them while the 96 MFMAs of the current ones run: 56 VALU
    // instructions per fragment (second operand 48), five or six in the shadow of each
    // MFMA.  (Residuals by v_dot2_f32_bf16, 28 instructions, were slower: 207 TFLOP/s.)
    using frag16 = typename Mma<BF16>::frag;
    constexpr float kScale = 0x1p40f, kUnscale = 0x1p-40f;
    constexpr int kPl = 3, kFr = kTM + kTN;
    constexpr int kOpSlots = 11;  // slots a fragment's split takes
    constexpr int kSlots = 2 * kPl * kMB;            // MFMAs per 16 hidden elements
    constexpr int kOps = 52, kPer = 5;               // steps of a fragment's split, per slot
    constexpr int kFirst = kSlots - kFr * kOpSlots;  // slot of the first split op
    static_assert(kFirst >= 4 && kKK == 4, "reads ahead of the split");
    // the lane's 8 hidden elements 16 kk + 8 (lane / 32) + 0..7 of a row: two chunks
    int foff[2][2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int c = 0; c < 2; ++c) foff[kk][c] = lds_off(frow, kk * 4 + (lane >> 5) * 2 + c);
    frag16 pl[2][kFr][kPl];  // [set][A fragments, then B][plane]
    float raw[3][8];
    float h0, h1, r0, r1;
    uint32_t lost = 0;  // the third planes are the last residuals unless one has bits in its low half
    uint32_t out[kPl][4];
    auto read_raw = [&](const unsigned char* stage, int kk, int f) __attribute__((always_inline)) {
      const unsigned char* rows = f < kTM ? stage + (wm * kWM + f * 32) * kRowBytes
                                          : stage + kHalfBytes + (wn * kWN + (f - kTM) * 32) * kRowBytes;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const frag q = *reinterpret_cast<const frag*>(rows + foff[kk][c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[f % 3][c * 4 + e] = q[e];
      }
    };
    // op N of the split of fragment F into set SET
    auto split_op = [&](auto set_c, auto f_c, auto n_c) __attribute__((always_inline)) {
      constexpr int F = decltype(f_c)::value, N = decltype(n_c)::value;
      constexpr int P = N / 13, O = N % 13;
      float* x = raw[F % 3];
      if constexpr (O == 0) {
        if constexpr (F < kTM) {
          x[2 * P] *= kScale;
          x[2 * P + 1] *= kScale;
        }
      } else if constexpr (O == 1) out[0][P] = BF16::pack2(x[2 * P], x[2 * P + 1]);
      else if constexpr (O == 2) h0 = low_bf16(out[0][P]);
      else if constexpr (O == 3) h1 = __uint_as_float(out[0][P] & 0xffff0000u);
      else if constexpr (O == 4) r0 = x[2 * P] - h0;
      else if constexpr (O == 5) r1 = x[2 * P + 1] - h1;
      else if constexpr (O == 6) out[1][P] = BF16::pack2(r0, r1);
      else if constexpr (O == 7) h0 = low_bf16(out[1][P]);
      else if constexpr (O == 8) h1 = __uint_as_float(out[1][P] & 0xffff0000u);
      else if constexpr (O == 9) r0 = r0 - h0;
      else if constexpr (O == 10) r1 = r1 - h1;
      else if constexpr (O == 11) out[2][P] = BF16::pack2(r0, r1);
      else lost = or3(lost, r0, r1);
      if constexpr (N == kOps - 1) {
#pragma unroll
        for (int k = 0; k < kPl; ++k) {
          const vu4 q = {out[k][0], out[k][1], out[k][2], out[k][3]};
          pl[decltype(set_c)::value][F][k] = __builtin_bit_cast(frag16, q);
        }
      }
    };
    // One step: the 96 MFMAs of set SET (products a2 b0, a0 b2, a1 b1, a1 b0, a0 b1,
    // a0 b0 of the 16 tiles), beside them the reads and the split of the next 16
    // hidden elements (half kk of `stage`) into the other set, and with LOAD the
    // direct loads of stage data t_load into `into`.
    auto step16 = [&](auto set_c, const unsigned char* stage, int kk, auto load_c, unsigned char* into,
                      int t_load) __attribute__((always_inline)) {
      constexpr int SET = decltype(set_c)::value;
      constexpr bool LOAD = decltype(load_c)::value;
      static_for<kSlots>([&](auto q_c) __attribute__((always_inline)) {
        constexpr int Q = decltype(q_c)::value;
        constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
        constexpr int PR = Q / kMB, I = Q / kTN % kTM, J = Q % kTN;
        acc[I][J] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pl[SET][kTM + J][pb[PR]], pl[SET][I][pa[PR]],
                                                            acc[I][J], 0, 0, 0);
        // the first two fragments are read at once, each other one a split ahead
        if constexpr (Q == 0) read_raw(stage, kk, 0);
        if constexpr (Q == 2) read_raw(stage, kk, 1);
        if constexpr (Q >= kFirst) {
          constexpr int F = (Q - kFirst) / kOpSlots, N = (Q - kFirst) % kOpSlots * kPer;
          if constexpr (N == 0 && F + 2 < kFr) read_raw(stage, kk, F + 2);
          static_for<kPer>([&](auto u_c) __attribute__((always_inline)) {
            if constexpr (N + decltype(u_c)::value < kOps)
              split_op(std::integral_constant<int, SET ^ 1>{}, std::integral_constant<int, F>{},
                       std::integral_constant<int, N + decltype(u_c)::value>{});
          });
        }
        if constexpr (LOAD && Q % 4 == 1 && Q / 4 < kL) dma(into, t_load, Q / 4);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    // Prologue: stage data 0 and 1 in flight, the first 16 elements split.
#pragma unroll
    for (int q = 0; q < kL; ++q) dma(st0, 0, q);
#pragma unroll
    for (int q = 0; q < kL; ++q) dma(st1, 1, q);
    wait_vm_barrier<kL>();
    static_for<kFr>([&](auto f_c) __attribute__((always_inline)) {
      read_raw(st0, 0, decltype(f_c)::value);
      static_for<kOps>([&](auto n_c) __attribute__((always_inline)) { split_op(S0{}, f_c, n_c); });
    });
    // Stage t: step 0 computes its first half and splits its second; then every
    // wave has read the stage and, past the barrier, step 1 refills it with stage
    // data t + 2 while it splits the first half of stage t + 1.  Past the last
    // stage the loads and the split repeat the last stage's data, unused.
    auto stage2 = [&](int t, auto s_c) __attribute__((always_inline)) {
      constexpr int S = decltype(s_c)::value;
      unsigned char* cur = stage_ptr(S);
      step16(S0{}, cur, 1, F_{}, cur, 0);
      wait_vm_barrier<0>();
      step16(S1{}, stage_ptr(S ^ 1), 0, T_{}, cur, t + 2 < nst ? t + 2 : nst - 1);
    };
    for (int t = 0; t < nst; t += kStages) {
      stage2(t, S0{});
      stage2(t + 1, S1{});
    }
    wait_vm_barrier<0>();
    // Infinities and NaN do not split (inf - inf), nor does a value that the scale
    // takes to infinity or that rounds there as a bf16; a sum of 2^88 overflows under
    // the scale; and a second operand below 2^-109 can have bits that its planes do not
    // hold: a tile in which one shows is formed again with fp32 MFMAs.
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
      for (int j = 0; j < kTN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) z += acc[i][j][v] * 0.f;
    unscale = kUnscale;
    if (__syncthreads_or(!(z == 0.f) || (lost & 0xffffu) != 0)) {
      clear_acc();
      run_stages();
      unscale = 1.f;
    }
  } else {
    run_stages();
    if constexpr (kAdapters) {
      if constexpr (kF16) keep_acc();  // (on both sides of the branch, or 13 registers are spilled)
      if (apart) adapter_stages();
      if constexpr (kF16) keep_acc();
    }
  }

  if constexpr (MODE == kGemm) {
    // ---- plain GEMM: the accumulators go straight to C ----
    // a 16-bit output over an fp32 running sum adds C before it rounds
    const bool add_c = P.accumulate && P.C != nullptr;
    float* C = P.C == nullptr ? nullptr : P.C + ks * P.nrows * P.ldc;
    // each lane holds groups of four consecutive columns of a row, moved as one
    // 16-byte (fp32) or 8-byte (16-bit) piece where base and row stride allow.  One
    // unrolled loop per kind of store: a single loop choosing its store per element
    // grew past what the compiler unrolls and put the accumulators on the stack.
    const bool vec_c = C != nullptr && (reinterpret_cast<uintptr_t>(C) & 15u) == 0 && P.ldc % 4 == 0;
    const bool vec_b = P.Cb != nullptr && (reinterpret_cast<uintptr_t>(P.Cb) & 7u) == 0 && P.ldcb % 4 == 0;
    auto each = [&](auto&& put) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kTM; ++i) {
        const int64_t row = m0 + wm * kWM + i * kT + frow;
        if (row >= row_end) continue;
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
          for (int g = 0; g < kAV / 4; ++g) {
            const int64_t col = n0 + wn * kWN + j * kT + g * 8 + lane / kT * 4;
            f32x4 o = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            if constexpr (std::is_same<E, F32>::value) {
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] *= unscale;
            }
            if (col < P.V) put(row, col, o, col + 4 <= P.V);
          }
      }
    };
    auto load_c = [&](int64_t row, int64_t col, bool full) {
      const float* src = C + row * P.ldc + col;
      f32x4 c = {0.f, 0.f, 0.f, 0.f};
      if (full && vec_c) {
        c = *reinterpret_cast<const f32x4*>(src);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < P.V) c[e] = src[e];
      }
      return c;
    };
    auto store_c = [&](int64_t row, int64_t col, f32x4 o, bool full) {
      float* dst = C + row * P.ldc + col;
      if (full && vec_c) {
        *reinterpret_cast<f32x4*>(dst) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < P.V) dst[e] = o[e];
      }
    };
    auto store_b = [&](auto eb, int64_t row, int64_t col, f32x4 o, bool full) {
      using EB = decltype(eb);
      uint16_t* dst = P.Cb + row * P.ldcb + col;
      const uint2 w = pack4<EB>(o);
      if (full && vec_b) {
        *reinterpret_cast<uint2*>(dst) = w;
      } else {
        const uint32_t wv[2] = {w.x, w.y};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < P.V) dst[e] = (uint16_t)(wv[e >> 1] >> (16 * (e & 1)));
      }
    };
    auto out_b = [&](auto eb) __attribute__((always_inline)) {
      if (add_c)
        each([&](int64_t row, int64_t col, f32x4 o, bool full)
                 __attribute__((always_inline)) { store_b(eb, row, col, load_c(row, col, full) + o, full); });
      else
        each([&](int64_t row, int64_t col, f32x4 o, bool full)
                 __attribute__((always_inline)) { store_b(eb, row, col, o, full); });
    };
    constexpr bool k16 = !std::is_same<E, F32>::value;  // 16-bit outputs: 16-bit operands only
    if (k16 && to_bf16 && P.cb_f16) {
      if constexpr (k16) out_b(F16{});
    } else if (k16 && to_bf16) {
      if constexpr (k16) out_b(BF16{});
    } else if (add_c)
      each([&](int64_t row, int64_t col, f32x4 o, bool full)
               __attribute__((always_inline)) { store_c(row, col, load_c(row, col, full) + o, full); });
    else
      each([&](int64_t row, int64_t col, f32x4 o, bool full)
               __attribute__((always_inline)) { store_c(row, col, o, full); });
  } else if constexpr (MODE == kFwdX) {
    // ---- forward, logits in fp32: the rows are reduced in the registers ----
    //
    // e4m3 of [16384, 4096] x [151936, 4096]: 7.4 ms, 2.75 PFLOP/s (the library's product of
    // these operands, which writes the logits and has no log-sum-exp, 2.89); the MFMA units are
    // busy 68 to 71% of the cycles at the 1.6 to 1.7 GHz that this load leaves: bound by power.
    //
    // A lane holds kTN groups of columns of kTM rows, the lanes that share a row are kT apart
    // and the two waves of a row band exchange through LDS.
    wait_vm_barrier<0>();
    // (the accumulators are complete here: without this the compiler moves MFMAs of the last
    // stage down between the rows' reductions, and they wait for each other)
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
      for (int j = 0; j < kTN; ++j) asm volatile("" : "+a"(acc[i][j]));
    constexpr int kG = kAV / 4;  // groups of four consecutive columns per MFMA tile
    const int col_lane = lane / kT * 4;
    const int64_t ncols = P.V - n0;
    // A value is y with the logit x = y * rs: e4m3 products come with the column's scale, and the
    // row's goes into the exponent's factor, 2^(y c - M c) with c = rs log2(e), one fma a value.  The
    // rounding of M c is undone at the end.  (c is kept above 0, so that the columns past the end,
    // -inf, stay that under a row scale of 0; a negative row scale goes into the values.)
    // Row by row of MFMA tiles, so that each accumulator is read once.
    float rm[kTM], rsum[kTM];
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
      const int rl = wm * kWM + i * kT + frow;
      float rs = kES == 1 ? s_rs[rl] : 1.f;
      const float f = rs < 0.f ? rs : 1.f;
      rs = rs < 0.f ? 1.f : rs;
      const bool negative = kES == 1 && __ballot(f != 1.f) != 0;
      // few tiles hold a row's target: looked for only where one does
      const int tc = s_tcol[rl] - wn * kWN;
      const bool held = __ballot(tc >= 0 && tc < kWN) != 0;
      float y[kTN][kAV];
      float M = -INFINITY;
#pragma unroll
      for (int j = 0; j < kTN; ++j)
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          float c4[4] = {1.f, 1.f, 1.f, 1.f};
          if constexpr (kES == 1) {
            const float4 cs = *reinterpret_cast<const float4*>(s_ls + wn * kWN + j * kT + g * 8 + col_lane);
            c4[0] = cs.x;
            c4[1] = cs.y;
            c4[2] = cs.z;
            c4[3] = cs.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) y[j][4 * g + e] = kES == 1 ? acc[i][j][4 * g + e] * c4[e] : acc[i][j][4 * g + e];
        }
      if (negative) {
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
          for (int v = 0; v < kAV; ++v) y[j][v] *= f;
      }
      if (ncols < kBN) {
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
          for (int v = 0; v < kAV; ++v)
            if (wn * kWN + j * kT + v / 4 * 8 + col_lane + v % 4 >= ncols) y[j][v] = -INFINITY;
      }
      if (held) {
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
          for (int v = 0; v < kAV; ++v)
            if (j * kT + v / 4 * 8 + col_lane + v % 4 == tc) P.xt[m0 + rl - P.row0] = y[j][v] * rs;
      }
#pragma unroll
      for (int j = 0; j < kTN; ++j)
#pragma unroll
        for (int v = 0; v < kAV; ++v) M = fmaxf(M, y[j][v]);
#pragma unroll
      for (int off = kT; off < kWave; off <<= 1) M = fmaxf(M, __shfl_xor(M, off, kWave));
      const float c = kES == 1 ? fmaxf(rs * kLog2e, 0x1p-126f) : kLog2e, Mc = M * c;
      float s4[4] = {0.f, 0.f, 0.f, 0.f};
      if (M != -INFINITY) {
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
          for (int v = 0; v < kAV; ++v) s4[v & 3] += fast_exp2(fmaf(y[j][v], c, -Mc));
      } else {  // columns that are not there, -inf and NaN, which a maximum does not show
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
          for (int v = 0; v < kAV; ++v) s4[v & 3] = y[j][v] != y[j][v] ? y[j][v] : s4[v & 3];
      }
      float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
      for (int off = kT; off < kWave; off <<= 1) sum += __shfl_xor(sum, off, kWave);
      if (M != -INFINITY) {  // (else the sum is 0 or NaN)
        sum *= fast_exp2(-fmaf(M, c, -Mc));
        M = kES == 1 ? M * rs : M;
      }
      rm[i] = M;
      rsum[i] = sum;
      if (wn == 1 && lane < kT) {
        s_m[rl] = M;
        s_g[rl] = sum;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    if (wn == 0 && lane < kT) {
#pragma unroll
      for (int i = 0; i < kTM; ++i) {
        const int rl = wm * kWM + i * kT + frow;
        const int64_t r = m0 + rl;
        if (r >= row_end) continue;
        const float m1 = s_m[rl], M = fmaxf(rm[i], m1);
        float sum = 0.f;
        if (counts(rm[i], rsum[i])) sum += rsum[i] * fast_exp2((rm[i] - M) * kLog2e);
        if (counts(m1, s_g[rl])) sum += s_g[rl] * fast_exp2((m1 - M) * kLog2e);
        if constexpr (kAdapters) {
          if (n_seg > 0 && s_ord[rl] >= 0 && (s_bad[s_ord[rl]] & kBroken) != 0) sum = __builtin_nanf("");
        }
        float* dst = P.part + ((r - P.row0) * P.n_nt + nt) * 2;
        dst[0] = M;
        dst[1] = sum;
      }
    }
  } else {
  // ---- epilogue: the tile goes through LDS as bf16, one row per thread ----
  //
  // The accumulators of a row are spread over lanes and waves; instead of cross-lane
  // reductions each wave writes its quarter to LDS (row-major [256][256] bf16
  // over the two stage arrays, 16-byte chunks XOR-swizzled by row; each lane
  // four consecutive columns of a row at a time) and thread t then walks row t
  // (forward) or copies rows out with 16-byte stores (gradient).  Every direct load
  // has landed (the last wait was vmcnt(0)); the barrier orders every wave's last
  // fragment reads before the stores.
  wait_vm_barrier<0>();
  const int wm_u = wave_u >> 1;
  const int col_lane = (lane >> 4) * 4;  // the lane's first column of an MFMA tile
  // the epilogue rows of this wave's quarter live in stage array wm
  uint16_t* const xq = reinterpret_cast<uint16_t*>(stage_ptr(wm_u));
  if (MODE == kFwd) {
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
      const int rl = wm * kWM + i * kT + frow;
#pragma unroll
      for (int j = 0; j < kTN; ++j)
        *reinterpret_cast<uint2*>(xq + xs_index(rl, wn * kWN + j * kT + col_lane)) = pack4<E>(acc[i][j]);
    }
    __syncthreads();
    const int64_t r = m0 + tid;
    if (r < row_end) {
      // row tid is local row tid % 128 of stage array tid / 128
      const uint16_t* xs = reinterpret_cast<const uint16_t*>(stage_ptr(wm_u));
      const int ncols = (P.V - n0 < kBN) ? (int)(P.V - n0) : kBN;
      const vu4* rowp = reinterpret_cast<const vu4*>(xs + (tid & (kEpiRows - 1)) * kBN);
      const int sw = xs_swizzle(tid);
      float M = -INFINITY, sum = 0.f;
      // two passes (max, then sum of exp); the column bound is only checked in
      // the last, partial column tile
      auto walk = [&](auto full_c) {
        constexpr bool FULL = decltype(full_c)::value;
        for (int c = 0; c < kBN / 8; ++c) {
          float w[8];
          E::unpack(rowp[c ^ sw], w);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (FULL || c * 8 + e < ncols) M = fmaxf(M, w[e]);
        }
        if (M != -INFINITY) {
          float s4[4] = {0.f, 0.f, 0.f, 0.f};
          for (int c = 0; c < kBN / 8; ++c) {
            float w[8];
            E::unpack(rowp[c ^ sw], w);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (FULL || c * 8 + e < ncols) s4[e & 3] += fast_exp2((w[e] - M) * kLog2e);
          }
          sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
        } else {  // -inf and NaN, which a maximum does not show
          for (int c = 0; c < kBN / 8; ++c) {
            float w[8];
            E::unpack(rowp[c ^ sw], w);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if ((FULL || c * 8 + e < ncols) && w[e] != w[e]) sum = w[e];
          }
        }
      };
      if (ncols == kBN)
        walk(std::true_type{});
      else
        walk(std::false_type{});
      float* dst = P.part + ((r - P.row0) * P.n_nt + nt) * 2;
      dst[0] = M;
      dst[1] = sum;
      const int tc = s_tcol[tid];
      if (tc >= 0) P.xt[r - P.row0] = value_of<E>(xs[xs_index(tid, tc)]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
      const int rl = wm * kWM + i * kT + frow;
      const float gv = s_g[rl], M = s_m[rl], LS = s_ls[rl];
      const float off = (M + LS) * kLog2e;
      const int tc = s_tcol[rl];
#pragma unroll
      for (int j = 0; j < kTN; ++j) {
        const int cl = wn * kWN + j * kT + col_lane;
        f32x4 o;
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float x0 = acc[i][j][e], x1 = acc[i][j][e + 1];
          if constexpr (MODE == kGradX) {
            // (the offset's rounding moves a row's probabilities by 2^-24 |M + LS|, relatively)
            o[e] = fast_exp2(fmaf(x0, kLog2e, -off));
            o[e + 1] = fast_exp2(fmaf(x1, kLog2e, -off));
          } else {
            round_trip2<E>(x0, x1);  // the logits in the operand dtype
            o[e] = fast_exp2(((x0 - M) - LS) * kLog2e);
            o[e + 1] = fast_exp2(((x1 - M) - LS) * kLog2e);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (cl + e == tc) ? (1.f - o[e]) * gv : -o[e] * gv;
        // kGrad: G is bf16 for either operand dtype
        *reinterpret_cast<uint2*>(xq + xs_index(rl, cl)) =
            pack4<typename std::conditional<MODE == kGradX, E, BF16>::type>(o);
      }
    }
    __syncthreads();
    // 32 threads per row, one 16-byte chunk each; 8 rows per pass
    const int c = tid & 31;
#pragma unroll 4
    for (int k = 0; k < kBM / 8; ++k) {
      const int rl = (tid >> 5) + 8 * k;
      const int64_t r = m0 + rl;
      const int64_t col0 = n0 + c * 8;
      if (r >= row_end || col0 >= P.V) continue;
      const uint16_t* xs = reinterpret_cast<const uint16_t*>(stage_ptr(rl / kEpiRows));
      const vu4 q = reinterpret_cast<const vu4*>(xs + (rl & (kEpiRows - 1)) * kBN)[c ^ xs_swizzle(rl)];
      uint16_t* dst = P.G + (r - P.row0) * P.ldg + col0;
      if (col0 + 8 <= P.V && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
        *reinterpret_cast<vu4*>(dst) = q;
      } else {
        const uint32_t wv[4] = {q.x, q.y, q.z, q.w};
        for (int e = 0; e < 8 && col0 + e < P.V; ++e)
          dst[e] = (uint16_t)(wv[e >> 1] >> ((e & 1) * 16));
      }
    }
    if (P.Gt != nullptr) {
      // the transposed tile (rows of G past its end are zeros, which the caller's
      // padded reduction length relies on): a wave takes 16 columns x 64 rows at a time,
      // lane l the column pair l % 8 and the eight rows from 8 (l / 8) on, so that eight
      // lanes store one 128-byte line of G^T (one column per lane, 64 lines open per
      // store, took 0.6-0.7 ms of 6.8 on [5888, 4096] x [151808, 4096]; this takes 0.3 of 6.1)
#pragma unroll 2
      for (int it = 0; it < kBN / 16 * (kBM / 64) / kWaves; ++it) {
        const int q = wave_u * (kBN / 16 * (kBM / 64) / kWaves) + it;
        const int cl = (q % (kBN / 16)) * 16 + (lane & 7) * 2;
        const int rl = (q / (kBN / 16)) * 64 + (lane >> 3) * 8;
        const int64_t col = n0 + cl;
        if (col >= P.V) continue;
        const uint16_t* xs = reinterpret_cast<const uint16_t*>(stage_ptr(rl / kEpiRows));
        uint16_t* dst = P.Gt + col * P.ldgt + (m0 - P.row0) + rl;
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // two rows' pairs of columns -> two columns' pairs of rows
          const uint32_t a = *reinterpret_cast<const uint32_t*>(xs + xs_index(rl + 2 * e, cl));
          const uint32_t b = *reinterpret_cast<const uint32_t*>(xs + xs_index(rl + 2 * e + 1, cl));
          lo[e] = (a & 0xffffu) | (b << 16);
          hi[e] = (a >> 16) | (b & 0xffff0000u);
        }
        *reinterpret_cast<vu4*>(dst) = vu4{lo[0], lo[1], lo[2], lo[3]};
        if (col + 1 < P.V) *reinterpret_cast<vu4*>(dst + P.ldgt) = vu4{hi[0], hi[1], hi[2], hi[3]};
      }
    }
  }
  }  // the fused epilogues
}

// ---------------------------------------------------------------------------
// few rows (kFwdX): 64 rows x 128 columns per workgroup
// ---------------------------------------------------------------------------
// With few rows the forward is bound by reading W once, and a 256-row tile spends its time on
// rows that are not there.  Here a stage is 64 rows of H (from L2) and 128 of W, three stages
// of 24 KB in a ring with two in flight, two workgroups a CU: 64 KB of W on the way to each CU.
// Wave w owns columns 32 w .. 32 w + 31 of the 64 rows.  64 rows, H = 4096, V = 151936: 225 us of
// the kernel with 16 adapters in bf16 (1.32 GB, 5.9 TB/s; the 256-row tile 347), 110 in e4m3
// (623 MB, 5.7 TB/s; 160).
constexpr int kRM = 64, kRN = 128, kRStages = 3;
constexpr int kRStageBytes = (kRM + kRN) * kRowBytes;          // 24 KB: the H rows, then W's
constexpr int kRLoadsA = kRM / kDmaRows / kWaves, kRLoadsB = kRN / kDmaRows / kWaves;  // per wave and stage
static_assert(kRLoadsB % 2 == 0 && kDmaPerWave % 2 == 0, "a load's parity among the wave's is that of its rows' eights");

template <class E, bool RAGGED>
__global__ __launch_bounds__(kThreads, 2) void lce_rows_kernel(LceParams P) {
  using frag = typename Mma<E>::frag;
  using acc_t = typename Mma<E>::acc_t;
  constexpr int kT = Mma<E>::kT, kTM = kRM / kT, kTN = kRN / kWaves / kT, kAV = kT * kT / kWave;
  constexpr int kES = (int)sizeof(typename E::raw), kSKE = kRowBytes / kES;
  constexpr int kFC = (int)sizeof(frag) / 16;
  constexpr int kKK = kRowBytes / (kWave / kT * (int)sizeof(frag));
  constexpr bool kAdapters = kES == 2, kF16 = std::is_same<E, F16>::value;
  const int ur = kF16 ? kURow<F16> : P.planes;
  constexpr int kOut = -0x7fffffff - 1;  // an offset out of range: reads as zero
  __shared__ __align__(1024) unsigned char st0[kRStageBytes];
  __shared__ __align__(1024) unsigned char st1[kRStageBytes];
  __shared__ __align__(1024) unsigned char st2[kRStageBytes];
  __shared__ int s_tcol[kRM], s_ord[kRM], s_seg[kRM], s_bad[kRM];
  __shared__ float s_rs[kRM], s_m[kWaves][kRM], s_sum[kWaves][kRM];
  __shared__ __align__(16) float s_cs[kES == 1 ? kRN : 4];
  auto stage_ptr = [&](int s) -> unsigned char* { return s == 0 ? st0 : s == 1 ? st1 : st2; };

  // one XCD takes neighbouring column tiles, all row tiles of one after the other
  const int64_t n_mt = (P.nrows + kRM - 1) / kRM, n_nt = (P.V + kRN - 1) / kRN, ntiles = n_mt * n_nt;
  const int64_t per_xcd = (ntiles + kXcds - 1) / kXcds;
  const int64_t gi = (int64_t)(blockIdx.x % kXcds) * per_xcd + blockIdx.x / kXcds;
  if ((int64_t)(blockIdx.x / kXcds) >= per_xcd || gi >= ntiles) return;
  const int64_t nt = uniform(gi / n_mt), mt = uniform(gi - gi / n_mt * n_mt);
  const int64_t m0 = mt * kRM, n0 = nt * kRN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const int a_rows = (int)(P.nrows - m0 < kRM ? P.nrows - m0 : kRM);
  const int b_rows = (int)(P.V - n0 < kRN ? P.V - n0 : kRN);

  int n_seg = 0;
  bool apart = false;
  if (wave == 0) {
    const int64_t r = m0 + lane;
    int tc = -1, a = -1, before = -1;
    if (lane < a_rows) {
      const int64_t s = r / P.bsz, b = r - s * P.bsz;
      const int64_t t = P.target[b * P.tsb + s * P.tss];
      if (!((t < P.vs) || (t >= P.ve) || (t - P.vs >= P.V))) {
        const int64_t c = t - P.vs - n0;
        if (c >= 0 && c < kRN) tc = (int)c;
      }
      if constexpr (kAdapters) {
        a = P.aid[r];
        before = lane > 0 ? P.aid[r - 1] : -1;
      }
      if constexpr (kES == 1) s_rs[lane] = P.row_scale[r];
    } else if constexpr (kES == 1) {
      s_rs[lane] = 0.f;
    }
    s_tcol[lane] = tc;
    if constexpr (kAdapters) {
      const bool head = a >= 0 && (lane == 0 || a != before);
      const uint64_t heads = __ballot(head);
      const int at = (int)__popcll(heads & (~0ull >> (63 - lane)));  // heads up to this row
      s_ord[lane] = a >= 0 ? at - 1 : -1;
      if (head) {
        s_seg[at - 1] = a;
        s_bad[at - 1] = P.bad[a];
      }
      if (lane == 0) s_m[0][0] = __int_as_float((int)__popcll(heads));
    }
  }
  if constexpr (kES == 1) {
    if (tid >= kWave && tid - kWave < kRN) s_cs[tid - kWave] = tid - kWave < b_rows ? P.col_scale[n0 + tid - kWave] : 0.f;
  }
  __syncthreads();
  if constexpr (kAdapters) {
    n_seg = __builtin_amdgcn_readfirstlane(__float_as_int(s_m[0][0]));
    apart = __builtin_amdgcn_readfirstlane(__syncthreads_or(tid < n_seg && s_bad[tid] != 0)) != 0 ||
            P.b_bytes >= (int64_t(1) << 31);
  }

  const int nst = (int)(P.Hd / kSKE);
  const int cpp = kAdapters ? P.r8 >> 3 : 1, cps = kAdapters ? P.planes * cpp : 1;
  const int n_ext = (n_seg * cps + 7) >> 3;
  const int total = apart ? nst : nst + n_ext;
  __amdgpu_buffer_rsrc_t rsrc_a = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(P.h) + m0 * P.ldh * kES), 0, (int)(a_rows * P.ldh * kES), 0x00020000);
  __amdgpu_buffer_rsrc_t rsrc_b = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(P.w) + n0 * P.ldw * kES), 0, (int)(b_rows * P.ldw * kES), 0x00020000);
  int voff_a[kRLoadsA], voff_b[kRLoadsB];
#pragma unroll
  for (int i = 0; i < kRLoadsA; ++i) {
    const int row = (wave * kRLoadsA + i) * kDmaRows + (lane >> 3);
    voff_a[i] = (int)(row * P.ldh * kES) + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
  }
#pragma unroll
  for (int i = 0; i < kRLoadsB; ++i) {
    const int row = (wave * kRLoadsB + i) * kDmaRows + (lane >> 3);
    voff_b[i] = (int)(row * P.ldw * kES) + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
  }
  // the loads of stage data t (past the last one: zeros, so that the count in flight stays)
  auto dma = [&](unsigned char* stage, int t) __attribute__((always_inline)) {
    const int soff = t < nst ? t * kRowBytes : 0;
#pragma unroll
    for (int i = 0; i < kRLoadsA; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_a, (lds_ptr_t)(stage + (wave_u * kRLoadsA + i) * kDmaBytes), 16,
                                               voff_a[i], soff, 0, 0);
#pragma unroll
    for (int i = 0; i < kRLoadsB; ++i) {
      int off = voff_b[i];
      if constexpr (RAGGED) {  // past W's row (see lce_tile_kernel)
        const int left = t < nst ? (int)(P.Hw * kES) - t * kRowBytes : kRowBytes;
        off = ((lane & 7) ^ (((lane >> 4) + 4 * (i & 1)) & 7)) * 16 >= left ? kOut : off;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc_b, (lds_ptr_t)(stage + kRM * kRowBytes + (wave_u * kRLoadsB + i) * kDmaBytes), 16, off, soff, 0, 0);
    }
  };
  // offsets of stage data t >= nst (see lce_tile_kernel)
  auto prepare = [&](int t) __attribute__((always_inline)) {
    if constexpr (kAdapters) {
      rsrc_a = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(P.U + m0 * (int64_t)(ur * P.r8)), 0,
                                                 a_rows * ur * P.r8 * 2, 0x00020000);
      // (apart: the loop reads nothing of B, which may hold anything and, past 2 GiB, kOut too)
      rsrc_b = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(P.B + n0 * P.r8), 0,
                                                 apart ? 0 : (int)(P.b_bytes - n0 * P.r8 * 2), 0x00020000);
    }
    auto place = [&](int row, int& seg, int& rem) {
      const int x = (t - nst) * 8 + ((lane & 7) ^ ((row >> 1) & 7));
      seg = x / cps;
      rem = x - seg * cps;
    };
#pragma unroll
    for (int i = 0; i < kRLoadsA; ++i) {
      const int row = (wave * kRLoadsA + i) * kDmaRows + (lane >> 3);
      int seg, rem;
      place(row, seg, rem);
      voff_a[i] = kAdapters && t < total && s_ord[row] == seg ? (row * ur * P.r8 + rem * 8) * 2 : kOut;
    }
#pragma unroll
    for (int i = 0; i < kRLoadsB; ++i) {
      const int row = (wave * kRLoadsB + i) * kDmaRows + (lane >> 3);
      int seg, rem;
      place(row, seg, rem);
      voff_b[i] = kAdapters && t < total && seg < n_seg && row < b_rows
                      ? (s_seg[seg] * (int)P.V * P.r8 + rem % cpp * 8 + row * P.r8) * 2
                      : kOut;
    }
  };

  const int frow = lane & (kT - 1);
  int frag_off[kKK];
#pragma unroll
  for (int kk = 0; kk < kKK; ++kk) frag_off[kk] = lds_off(frow, (kk * (kWave / kT) + lane / kT) * kFC);
  acc_t acc[kTM][kTN];
#pragma unroll
  for (int i = 0; i < kTM; ++i)
#pragma unroll
    for (int j = 0; j < kTN; ++j)
#pragma unroll
      for (int v = 0; v < kAV; ++v) acc[i][j][v] = 0.f;
  auto fread = [&](const unsigned char* base, int kk) __attribute__((always_inline)) {
    if constexpr (kFC == 1) {
      return *reinterpret_cast<const frag*>(base + frag_off[kk]);
    } else {
      const vu4 a = *reinterpret_cast<const vu4*>(base + frag_off[kk]);
      const vu4 b = *reinterpret_cast<const vu4*>(base + (frag_off[kk] ^ 16));
      return frag{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    }
  };
  auto compute = [&](const unsigned char* stage) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) {
      frag fa[kTM], fb[kTN];
#pragma unroll
      for (int j = 0; j < kTN; ++j) fb[j] = fread(stage + (kRM + wave * (kRN / kWaves) + j * kT) * kRowBytes, kk);
#pragma unroll
      for (int i = 0; i < kTM; ++i) fa[i] = fread(stage + i * kT * kRowBytes, kk);
#pragma unroll
      for (int i = 0; i < kTM; ++i)
#pragma unroll
        for (int j = 0; j < kTN; ++j) acc[i][j] = Mma<E>::run(fb[j], fa[i], acc[i][j]);
    }
  };
  // Stage t: this wave's loads of it have landed when only those of t + 1 are in flight; past
  // the barrier everyone's have, and everyone has read stage t - 1, whose place t + 2 takes.
  auto step = [&](int t, auto s_c) __attribute__((always_inline)) {
    constexpr int S = decltype(s_c)::value;
    if (t + 2 >= nst) prepare(t + 2);
    wait_vm_barrier<kRLoadsA + kRLoadsB>();
    dma(stage_ptr((S + 2) % kRStages), t + 2);
    compute(stage_ptr(S));
  };
  dma(st0, 0);
  dma(st1, 1);
  for (int t = 0; t < total; t += kRStages) {
    step(t, std::integral_constant<int, 0>{});
    step(t + 1, std::integral_constant<int, 1>{});
    step(t + 2, std::integral_constant<int, 2>{});
  }
  wait_vm_barrier<0>();
  if constexpr (kAdapters) {
    // an adapter holds a value that is none (its rows become NaN, the others must not meet it),
    // B passes 2 GiB or a row's U fp16's range: the adapters' part by itself (see lce_tile_kernel)
    if (apart) {
      bool wide = false;
      auto scale_rows = [&](bool back) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kTM; ++i) {
          float f = s_rs[i * kT + frow];
          f = back ? 1.f / f : f;
#pragma unroll
          for (int j = 0; j < kTN; ++j)
#pragma unroll
            for (int v = 0; v < kAV; ++v) acc[i][j][v] *= f;
        }
      };
      if constexpr (kF16) {
        const bool mine = tid < kRM && s_ord[tid] >= 0 && (s_bad[s_ord[tid]] & kWide) != 0;
        if (tid < kRM) s_rs[tid] = mine ? wide_scale(u_f32(P.U, m0 + tid, P.r8), P.r8) : 1.f;
        wide = __syncthreads_or(mine) != 0;
        if (wide) scale_rows(false);
      }
      for (int e = 0; e < n_ext; ++e) {
        const int chunk = tid & 7, x = e * 8 + chunk, q = x / cps, rem = x - q * cps;
        const bool any = q < n_seg;
        const uint16_t* bp = P.B + ((int64_t)(any ? s_seg[q] : 0) * P.V + n0) * P.r8 + rem % cpp * 8;
        constexpr uint32_t ex = std::is_same<E, BF16>::value ? 0x7f80u : 0x7c00u;
        for (int row = tid >> 3; row < kRN; row += kThreads / 8) {
          vu4 u = {0u, 0u, 0u, 0u}, b = {0u, 0u, 0u, 0u};
          if (any && row < b_rows) b = *reinterpret_cast<const vu4*>(bp + (int64_t)row * P.r8);
          bool none = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) none |= (b[j] & ex) == ex || ((b[j] >> 16) & ex) == ex;
          if (none) b = vu4{0u, 0u, 0u, 0u};
          *reinterpret_cast<vu4*>(st0 + kRM * kRowBytes + lds_off(row, chunk)) = b;
          if (row < kRM) {
            if (any && s_ord[row] == q) {
              u = *reinterpret_cast<const vu4*>(P.U + (m0 + row) * (int64_t)(ur * P.r8) + rem * 8);
              if constexpr (kF16) {
                if (wide) u = plane8<E>(u_f32(P.U, m0 + row, P.r8) + rem % cpp * 8, s_rs[row], rem / cpp);
              }
            }
            *reinterpret_cast<vu4*>(st0 + lds_off(row, chunk)) = u;
          }
        }
        __syncthreads();
        compute(st0);
        __syncthreads();
      }
      if constexpr (kF16) {
        if (wide) scale_rows(true);
      }
    }
  }

  // ---- epilogue: the rows reduced in the registers, the four waves joined through LDS ----
  const int col_lane = lane / kT * 4;
#pragma unroll
  for (int i = 0; i < kTM; ++i) {
    const int rl = i * kT + frow, tc = s_tcol[rl] - wave * (kRN / kWaves);
    float M = -INFINITY;
#pragma unroll
    for (int j = 0; j < kTN; ++j)
#pragma unroll
      for (int v = 0; v < kAV; ++v) {
        const int c = j * kT + v / 4 * 8 + col_lane + v % 4;
        float x = acc[i][j][v];
        if constexpr (kES == 1) x = (x * s_cs[wave * (kRN / kWaves) + c]) * s_rs[rl];
        if (wave * (kRN / kWaves) + c >= b_rows) x = -INFINITY;
        if (c == tc) P.xt[m0 + rl] = x;
        acc[i][j][v] = x;
        M = fmaxf(M, x);
      }
#pragma unroll
    for (int off = kT; off < kWave; off <<= 1) M = fmaxf(M, __shfl_xor(M, off, kWave));
    float sum = 0.f;
    if (M != -INFINITY) {
#pragma unroll
      for (int j = 0; j < kTN; ++j)
#pragma unroll
        for (int v = 0; v < kAV; ++v) sum += fast_exp2((acc[i][j][v] - M) * kLog2e);
    } else {  // (see lce_tile_kernel)
#pragma unroll
      for (int j = 0; j < kTN; ++j)
#pragma unroll
        for (int v = 0; v < kAV; ++v) sum = acc[i][j][v] != acc[i][j][v] ? acc[i][j][v] : sum;
    }
#pragma unroll
    for (int off = kT; off < kWave; off <<= 1) sum += __shfl_xor(sum, off, kWave);
    if (lane < kT) {
      s_m[wave][rl] = M;
      s_sum[wave][rl] = sum;
    }
  }
  __syncthreads();
  if (tid < a_rows) {
    float M = s_m[0][tid], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w][tid]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (counts(s_m[w][tid], s_sum[w][tid])) sum += s_sum[w][tid] * fast_exp2((s_m[w][tid] - M) * kLog2e);
    if constexpr (kAdapters) {
      if (s_ord[tid] >= 0 && (s_bad[s_ord[tid]] & kBroken) != 0) sum = __builtin_nanf("");
    }
    float* dst = P.part + ((m0 + tid) * n_nt + nt) * 2;
    dst[0] = M;
    dst[1] = sum;
  }
}

// The maximum M and the sum of exponentials s of a row from its n partial pairs, by the W waves
// that share it (W == 1: all lanes of one wave; W == 4: the workgroup, which has one row).
template <int W>
__device__ __forceinline__ void join_partials(const float* __restrict__ p, int64_t n, float& M, float& s) {
  __shared__ float s_j[2][W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t first = W == 1 ? lane : threadIdx.x;
  M = -INFINITY;
#pragma unroll 4
  for (int64_t j = first; j < n; j += 64 * W) M = fmaxf(M, p[2 * j]);
  M = wave_max(M);
  if constexpr (W > 1) {
    if (lane == 0) s_j[0][wave] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, s_j[0][w]);
  }
  s = 0.f;
#pragma unroll 4
  for (int64_t j = first; j < n; j += 64 * W) {
    const float mj = p[2 * j], sj = p[2 * j + 1];
    if (counts(mj, sj)) s += sj * fast_exp2((mj - M) * kLog2e);
  }
  s = wave_sum(s);
  if constexpr (W > 1) {
    if (lane == 0) s_j[1][wave] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += s_j[1][w];
  }
}
// Rows up to which a workgroup joins one row's partials (17 us of [64, 1187] with one wave a
// row, 8 with four); more rows have waves enough.
constexpr int64_t kJoinRows = 2048;

// Per row: combine the column-tile partials into the row's max and log-sum-exp,
// then logprob = (x_t - max) - logsum (0 for targets outside the slice).
// W waves per row; with `perm` the partials' row r is row perm[r] of targets and results.
template <int W>
__global__ __launch_bounds__(256) void lce_merge_kernel(
    const float* __restrict__ part, const float* __restrict__ xt, int64_t row0, int64_t nrows,
    int64_t n_nt, int64_t bsz, const int64_t* __restrict__ target, int64_t tsb, int64_t tss,
    int64_t vs, int64_t ve, int64_t V, float* __restrict__ out, int64_t osb, int64_t oss,
    float* __restrict__ stats, const int64_t* __restrict__ perm) {
  const int64_t rl = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (rl >= nrows) return;
  float M, s;
  join_partials<W>(part + rl * n_nt * 2, n_nt, M, s);
  if ((threadIdx.x & (64 * W - 1)) == 0) {
    const int64_t r = perm != nullptr ? perm[row0 + rl] : row0 + rl;
    const int64_t sq = r / bsz, b = r - sq * bsz;
    const int64_t t = target[b * tsb + sq * tss];
    const bool tmask = (t < vs) || (t >= ve) || (t - vs >= V);
    const float logsum = logf(s);
    out[b * osb + sq * oss] = tmask ? 0.f : (xt[rl] - M) - logsum;
    if (stats != nullptr) {
      stats[2 * r] = M;
      stats[2 * r + 1] = logsum;
    }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Hd of LceParams for a weight whose rows hold Hw elements of `bytes` bytes: whole pairs of stages.
int64_t padded_hidden(int64_t Hw, int64_t bytes) {
  const int64_t pair = kStages * kRowBytes / bytes;
  return ceil_div(Hw, pair) * pair;
}

// The forward kernel with fp32 logits for T rows (P.part, P.xt not set yet: `workspace` holds
// mirl_lce_x_workspace_elems(T, V) floats).  Returns the number of tiles.
// Rows up to which lce_rows_kernel is taken.  Whole calls over [151936, 4096], 64-row tiles
// against 256-row ones, us: 64 rows 255 and 355 in bf16, 130 and 193 in e4m3; 128 rows 349 and
// 365, 171 and 186; 192 rows 434 and 394, 215 and 192.
constexpr int64_t kFewRows = 128;
template <class E>
int64_t launch_fwd_x(LceParams& P, float* workspace, hipStream_t st) {
  const bool few = P.nrows <= kFewRows;
  P.n_mt = ceil_div(P.nrows, few ? kRM : kBM);
  P.n_nt = ceil_div(P.V, few ? kRN : kBN);
  P.part = workspace;
  P.xt = workspace + P.nrows * P.n_nt * 2;
  const int64_t grid = ceil_div(P.n_mt * P.n_nt, kXcds) * kXcds;
  if (grid >= (int64_t(1) << 24)) return grid;  // a launch holds fewer than 2^32 threads
  const bool ragged = P.Hw != P.Hd;
  const auto kernel = few ? ragged ? lce_rows_kernel<E, true> : lce_rows_kernel<E, false>
                          : ragged ? lce_tile_kernel<kFwdX, E, true> : lce_tile_kernel<kFwdX, E, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kThreads), 0, st, P);
  return grid;
}

}  // namespace
}  // namespace mirl
