// Matrix products of rows with weight rows, dense and grouped by expert (no reference call site).
//   out[m][n] = sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b of 128} x[m][k] * w[n][k]      e4m3 operands, fp32 scales
//   out[m][n] = sum_k x[m][k] * w[n][k]                                                             bf16 / fp16 operands
// Grouped: rows [offsets[e], offsets[e + 1]) of the output take w[e]; the left rows may be gathered through an index.
//
// One K step is 128 bytes of a row: 128 e4m3 values = one scale block = ONE v_mfma_f32_16x16x128_f8f6f4 per 16 x 16 outputs,
// or 64 16-bit values = two v_mfma_f32_16x16x32.  The weights are the MFMA's first operand and the rows its second, so that a lane
// holds ONE row's outputs (column of D = lane & 15) and a row's scale is one register per lane: acc += (sx * sw) * partial is one
// multiply per 16 rows and step and four FMAs per MFMA.  The partial sum of a block starts from the MFMA's own zero, the sum
// over blocks stays in fp32 registers.
// Precision of the e4m3 MFMAs (both f8f6f4 and the older 16x16x32 form, measured with single products): 8 consecutive products
// are aligned to the one of largest exponent E and cut towards zero below 2^(E - 13); the groups of 8 are then added with 24 bits.  So an
// output is off by less than 2^-10 of the sum over groups of their largest |product| (seen: 2^-12), and by any part of itself where products
// cancel.  In the 2-norm over 2^20 outputs of 128 products it is 1.5e-5 of the result for normal operands, 5.3e-5 for heavy-tailed ones
// (normal * exp(1.5 normal)), 3.3e-6 for operands of one sign: far inside a bf16 or fp16 rounding, but not a 32-bit result.  For fp32 outputs (KIND_FP8_WIDE) the operands become bf16 in registers, which is exact, and a block is four v_mfma_f32_16x16x32_bf16:
// those keep 24 bits below the largest of 8 products (2^16 - 2^16 + 2^j keeps 2^j down to j = -8 in one group of 8), at half the matrix rate.
//
// matmul_kernel: tile BM rows x BN weight rows, both operands through LDS by LDS-DMA (16 bytes per lane, S stages of one K step).  LDS
// rows are 128 B; the 16-byte chunk index is XOR-swizzled on the source address so that the 16 rows x 4 chunks of a fragment read fall
// on different banks (counted: no conflicts).  A wave's 64 weight rows are dealt to its four MFMAs in runs of four (row 32 (f / 2) + 8 g +
// 4 (f % 2) + i is row 4 g + i of fragment f), so that a lane ends with two runs of 8 consecutive outputs of its row, and the four lanes
// of a row with 64 bytes side by side per store (runs of 16, two stores of half a 32-byte sector: 16384 x 4096 x 2048 130 -> 126 us,
// 4096 x 4096 x 1024 22.6 -> 20.9, 2048 x 2048 x 512 7.1 -> 6.5).
// matmul_few_kernel: small tiles whose K steps are dealt to the block's waves, each with an LDS ring of its own.
// Rows behind the last one are read from the last one and not stored.  A K step that ends inside its 128 bytes: chunks behind the
// row's end are read from the row's start and cleared before use, whatever they hold.
#include "common.h"
#include <algorithm>
#include <cmath>
#include <iterator>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(1))) void* gbl_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;
#ifdef __HIP_DEVICE_COMPILE__
typedef __amdgpu_buffer_rsrc_t buffer_t;
// raw buffer over everything behind a uniform pointer (its offsets are unsigned 32-bit)
__device__ __forceinline__ buffer_t make_buffer(const char* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0xffffffffu, 0x00027000);
}
#endif

enum { KIND_FP8 = 0, KIND_BF16 = 1, KIND_FP16 = 2, KIND_FP8_WIDE = 3 };
constexpr bool scaled(int kind) { return kind == KIND_FP8 || kind == KIND_FP8_WIDE; }

struct MatmulParams {
  const char* x;
  const char* w;
  const float* xs;
  const float* ws;
  const int32_t* rows;       // gather index of the left rows (NULL: row m)
  const int32_t* offsets;    // [E + 1] (NULL: one group of all rows)
  void* out;
  int64_t ldx, ldw, wstride; // bytes
  int64_t xs_m, xs_b, ldo;   // elements
  int64_t M, xrows;
  int N, Kb, nk, E, out_type;// Kb: bytes of a row that count; nk = ceil(Kb / 128)
  int mtiles_max, ntiles;
};

// One K step of a 16 x 16 tile: a and b hold a lane's 32 bytes of its weight row and of its row
template <int KIND>
__device__ __forceinline__ f32x4 mfma_step(const i32x8& a, const i32x8& b, f32x4 c) {
  if constexpr (KIND == KIND_FP8) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
  } else {
    const i32x4 a0 = __builtin_shufflevector(a, a, 0, 1, 2, 3), a1 = __builtin_shufflevector(a, a, 4, 5, 6, 7);
    const i32x4 b0 = __builtin_shufflevector(b, b, 0, 1, 2, 3), b1 = __builtin_shufflevector(b, b, 4, 5, 6, 7);
    if constexpr (KIND == KIND_BF16) {
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a0), __builtin_bit_cast(bf16x8, b0), c, 0, 0, 0);
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a1), __builtin_bit_cast(bf16x8, b1), c, 0, 0, 0);
    } else {
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a0), __builtin_bit_cast(f16x8, b0), c, 0, 0, 0);
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a1), __builtin_bit_cast(f16x8, b1), c, 0, 0, 0);
    }
  }
}
// 32 e4m3 values as bf16, and a K step of a 16 x 16 tile on two such operands
struct Wide {
  bf16x8 v[4];
};
__device__ __forceinline__ Wide widen(const i32x8& a) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  Wide r;
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[d], 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[d], 1.f, true);
    bf16x8& t = r.v[d >> 1];
    t[4 * (d & 1)] = lo[0], t[4 * (d & 1) + 1] = lo[1], t[4 * (d & 1) + 2] = hi[0], t[4 * (d & 1) + 3] = hi[1];
  }
  return r;
}
__device__ __forceinline__ f32x4 mfma_wide(const Wide& a, const Wide& b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ i32x8 read_pair(const char* lo, const char* hi) {
  return __builtin_shufflevector(*reinterpret_cast<const i32x4*>(lo), *reinterpret_cast<const i32x4*>(hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// the first n of the 16 bytes of v (n <= 0: none), the others zero
__device__ __forceinline__ i32x4 keep_bytes(i32x4 v, int n) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int k = n - 4 * d;
    v[d] = k >= 4 ? v[d] : k <= 0 ? 0 : v[d] & (int)((1u << (8 * k)) - 1u);
  }
  return v;
}

// the same for a lane's two chunks of a K step, n: bytes left from the first one on
__device__ __forceinline__ i32x8 keep_pair(i32x8 v, int n) {
  const i32x4 lo = keep_bytes(__builtin_shufflevector(v, v, 0, 1, 2, 3), n), hi = keep_bytes(__builtin_shufflevector(v, v, 4, 5, 6, 7), n - 64);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// chunk swizzles: eight different values over the 8 consecutive lanes' rows of a fragment read
__device__ __forceinline__ int swz_x(int row) { return row & 7; }
__device__ __forceinline__ int swz_w(int row) { return (row & 3) | ((row >> 3) & 1) << 2; }

// L consecutive outputs of a row to memory, in 16-byte stores of the element's alignment (the hardware takes any)
template <int L, typename T>
__device__ __forceinline__ void store_values(T* dst, const float* v, int n_left) {
  if (n_left >= L) {
    constexpr int S = L * sizeof(T) >= 16 ? 16 / sizeof(T) : L;      // elements per store
    typedef T txs __attribute__((ext_vector_type(S), aligned(sizeof(T))));
#pragma unroll
    for (int i = 0; i < L / S; ++i) {
      txs t;
#pragma unroll
      for (int e = 0; e < S; ++e) t[e] = (T)v[S * i + e];
      *reinterpret_cast<txs*>(dst + S * i) = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i < n_left) dst[i] = (T)v[i];
  }
}
template <int L>
__device__ __forceinline__ void store_run(void* out, int type, int64_t at, const float* v, int n_left) {
  if (type == DIGA_BF16) store_values<L>(static_cast<__bf16*>(out) + at, v, n_left);
  else if (type == DIGA_FP16) store_values<L>(static_cast<_Float16*>(out) + at, v, n_left);
  else store_values<L>(static_cast<float*>(out) + at, v, n_left);
}

// Ragged groups, scanned by every wave 64 at a time.  An offset below one before it counts as that one and none passes M, so
// groups never overlap and stay inside the output.
struct GroupScan {
  int lo, hi, tiles, upto;                                 // this lane's group: first row, end, tiles of BM rows, tiles up to and with it
  template <int BM>
  __device__ __forceinline__ void read(const int32_t* offsets, int E, int M, int e0, int run) {
    const int lane = threadIdx.x & 63, i = e0 + lane;
    lo = i <= E ? offsets[i] : 0, hi = i < E ? offsets[i + 1] : 0;
    lo = min(max(lo, run), M), hi = min(max(hi, run), M);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {                     // running maxima
      const int l = __shfl_up(lo, d), h = __shfl_up(hi, d);
      if (lane >= d) lo = max(lo, l), hi = max(hi, h);
    }
    hi = max(hi, lo);
    upto = tiles = i < E ? (hi - lo + BM - 1) / BM : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(upto, d);
      if (lane >= d) upto += u;
    }
  }
};

// The tile of this block: nt, and group e's rows m0 .. m1 (m0 the tile's first).  Blocks go round the 8 XCDs, so every XCD takes a
// contiguous range of the tiles, in bands of `band` row tiles: what runs together on an XCD shares rows and weight rows in its L2.
// False when there is no tile left (a grouped launch is sized for the worst split of M rows).
template <int BM, bool GROUPED>
__device__ __forceinline__ bool tile_of_block(const MatmulParams& p, int band, int& nt, int& e, int& m0, int& m1) {
  GroupScan g;
  int mtiles = p.mtiles_max, run = 0;
  if constexpr (GROUPED) {
    mtiles = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
      g.read<BM>(p.offsets, p.E, (int)p.M, e0, run);
      mtiles += __shfl(g.upto, 63), run = __shfl(g.hi, 63);
    }
    mtiles = __builtin_amdgcn_readfirstlane(mtiles);
  }
  const unsigned total = (unsigned)mtiles * (unsigned)p.ntiles, id = blockIdx.x;
  if (id >= total) return false;
  const unsigned xcd = id & 7, more = total & 7;
  const unsigned t = xcd * (total >> 3) + min(xcd, more) + (id >> 3);
  const unsigned width = (unsigned)min(band, mtiles) * (unsigned)p.ntiles, b = t / width, r = t - b * width;
  const unsigned high = min((unsigned)min(band, mtiles), (unsigned)mtiles - b * (unsigned)min(band, mtiles));
  nt = r / high;
  const int mt = b * min(band, mtiles) + (r - nt * high);
  if constexpr (!GROUPED) {
    e = 0, m0 = mt * BM, m1 = (int)p.M;
  } else {
    int before = 0;
    run = 0;
    for (int e0 = 0;; e0 += 64) {                          // (mt < mtiles: some chunk holds it)
      if (p.E > 64) g.read<BM>(p.offsets, p.E, (int)p.M, e0, run);
      const int here = __shfl(g.upto, 63);
      if (mt < before + here) {
        const int src = __ffsll(__ballot(g.upto > mt - before)) - 1;
        e = e0 + src;
        m0 = __shfl(g.lo, src) + (mt - before - __shfl(g.upto - g.tiles, src)) * BM;
        m1 = __shfl(g.hi, src);
        break;
      }
      before += here, run = __shfl(g.hi, 63);
    }
    e = __builtin_amdgcn_readfirstlane(e), m0 = __builtin_amdgcn_readfirstlane(m0), m1 = __builtin_amdgcn_readfirstlane(m1);
  }
  return true;
}

template <int KIND, int BM, int BN, int WM, int WN, int S, bool GROUPED>
__global__ __launch_bounds__(WM* WN * 64, 2) void matmul_kernel(MatmulParams p) {
#ifdef __HIP_DEVICE_COMPILE__                              // (the buffer type has no host form: a host pass over the body drops the launch stub)
  constexpr int NW = WM * WN;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;      // fragments per wave: rows, weight rows
  static_assert(TN == 4, "a wave's weight rows are dealt in runs of four over four fragments");
  static_assert(TM % 2 == 0, "row fragments take turns in two register sets; the last two fragments of a step run behind its barrier");
  constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW;        // LDS-DMA instructions (8 rows of 128 B) per wave and stage
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "every wave fills the same number of rows");
  static_assert(BM % 64 == 0 && BM / 64 < NW, "a wave loads 64 row scales or the weight scales");
  constexpr int SCALES = (BM + BN) * 128;                  // in a stage: x rows, w rows, x scales, w scales
  constexpr int STAGE = SCALES + (scaled(KIND) ? NW * 256 : 0);
  __shared__ __attribute__((aligned(1024))) char smem[S * STAGE];
  constexpr int PIECES = XI + WI + scaled(KIND);     // LDS-DMA instructions of a wave per stage
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 15, fg = lane >> 4;

  int nt, e, m0, m1;
  if (!tile_of_block<BM, GROUPED>(p, 8, nt, e, m0, m1)) return;
  const int n0 = nt * BN;
  auto source_row = [&](int row) -> int64_t {              // left row behind row `row` of the tile
    int64_t m = std::min(m0 + row, m1 - 1);
    if (GROUPED && p.rows) {
      m = p.rows[m];
      if (m < 0 || m >= p.xrows) m = 0;
    }
    return m;
  };

  // ---- sources of this lane's LDS-DMA pieces: LDS position (row, lane & 7) holds chunk (lane & 7) ^ swizzle(row)
  // Buffer loads with a uniform base (the tile's first row; x itself for gathered rows), constant 32-bit lane offsets and the K step
  // as scalar offset: no vector arithmetic per step.
  static_assert(NW % 4 == 0, "a lane's pieces all have the same swizzle");
  const int row0 = wave * 8 + (lane >> 3);
  const int xchunk = ((lane & 7) ^ swz_x(row0)) * 16, wchunk = ((lane & 7) ^ swz_w(row0)) * 16;   // of the piece inside a K step
  const int64_t xfirst = GROUPED && p.rows ? 0 : m0;
  const buffer_t xtile = make_buffer(p.x + xfirst * p.ldx);
  const buffer_t wtile = make_buffer(p.w + (int64_t)e * p.wstride + (int64_t)n0 * p.ldw);
  uint32_t xoff[XI], woff[WI];
#pragma unroll
  for (int i = 0; i < XI; ++i) xoff[i] = (uint32_t)((source_row(i * NW * 8 + row0) - xfirst) * p.ldx) + xchunk;
#pragma unroll
  for (int i = 0; i < WI; ++i) woff[i] = (uint32_t)(std::min(i * NW * 8 + row0, p.N - 1 - n0) * p.ldw) + wchunk;
  // scales, one 4-byte piece per lane: waves v < BM / 64 load those of rows 64 v ..., the others (all alike) one per 64 weight rows
  const float* ssrc = nullptr;
  int64_t sstep = 0;
  if constexpr (scaled(KIND)) {
    const int nb = (p.N + 127) >> 7;
    const bool of_rows = wave < BM / 64;
    ssrc = of_rows ? p.xs + source_row(wave * 64 + lane) * p.xs_m
                   : p.ws + ((int64_t)e * nb + std::min((n0 + std::min(lane, BN / 64 - 1) * 64) >> 7, nb - 1)) * p.nk;
    sstep = of_rows ? p.xs_b : 1;
  }
  const int whole = p.Kb >> 7;                             // K steps of 128 whole bytes
  auto fill_x = [&](int kb, int st, auto part) {           // part: the step may end inside its 128 bytes
    constexpr bool PART = decltype(part)::value;
    char* s = smem + st + wave * 1024;
    const int k0 = kb * 128;
    const bool xin = !PART || k0 + xchunk < p.Kb;
#pragma unroll
    for (int i = 0; i < XI; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xtile, (lds_ptr)(s + i * NW * 1024), 16, PART ? (xin ? xoff[i] + k0 : xoff[i] - xchunk) : xoff[i], PART ? 0 : k0, 0, 0);
    if constexpr (scaled(KIND)) __builtin_amdgcn_global_load_lds((gbl_ptr)(ssrc + kb * sstep), (lds_ptr)(smem + st + SCALES + wave * 256), 4, 0, 0);
  };
  auto fill_w = [&](int kb, int st, auto part) {
    constexpr bool PART = decltype(part)::value;
    char* s = smem + st + BM * 128 + wave * 1024;
    const int k0 = kb * 128;
    const bool win = !PART || k0 + wchunk < p.Kb;
#pragma unroll
    for (int i = 0; i < WI; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wtile, (lds_ptr)(s + i * NW * 1024), 16, PART ? (win ? woff[i] + k0 : woff[i] - wchunk) : woff[i], PART ? 0 : k0, 0, 0);
  };

  // the last K step may end inside its 128 bytes: what lies behind the row's end counts as zero
  auto clear_tail = [&](int st) {
    const int left = p.Kb - whole * 128;
    for (int t = tid; t < (BM + BN) * 8; t += NW * 64) {
      const int row = t >> 3, c = t & 7, keep = left - c * 16;
      const int sw = row < BM ? swz_x(row) : swz_w(row - BM);
      i32x4* q = reinterpret_cast<i32x4*>(smem + st + row * 128 + (c ^ sw) * 16);
      if (keep < 16) *q = keep_bytes(*q, keep);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int f = 0; f < TN; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};

  // fragment reads: lane (fr, fg) takes chunks fg and fg + 4 of its row
  const int wrow = wn * 64 + (fr >> 2) * 8 + (fr & 3);     // + 4 (f % 2) + 32 (f / 2): weight row of fragment f's row fr; the same swizzle for all f
  const char* wbase = smem + BM * 128 + wrow * 128;
  const char* xbase = smem + (wm * TM * 16 + fr) * 128;    // + 2048 i
  const int wofs[2] = {(fg ^ swz_w(wrow)) * 16, ((fg + 4) ^ swz_w(wrow)) * 16};
  const int xofs[2] = {(fg ^ swz_x(fr)) * 16, ((fg + 4) ^ swz_x(fr)) * 16};
  i32x8 w[TN], x[2];
  Wide ww[TN], xw;                                         // (KIND_FP8_WIDE)
  f32x4 part[2];
  float sx[2], s[2] = {0.f, 0.f}, sw = 0.f;
  auto read_w = [&](int st, int f) {
    const char* q = wbase + st + (f & 1) * 512 + (f >> 1) * 4096;
    w[f] = read_pair(q + wofs[0], q + wofs[1]);
  };
  auto read_x = [&](int st, int i, int slot) {
    x[slot] = read_pair(xbase + st + i * 2048 + xofs[0], xbase + st + i * 2048 + xofs[1]);
    if constexpr (scaled(KIND)) sx[slot] = *reinterpret_cast<const float*>(smem + st + SCALES + ((wm * TM + i) * 16 + fr) * 4);
  };
  auto read_sw = [&](int st) {
    return scaled(KIND) ? *reinterpret_cast<const float*>(smem + st + SCALES + BM * 4 + wn * 4) : 0.f;
  };
  // MFMA number n = i * TN + f of a step, and the FMAs that add the partial result of number n (by its block's scale)
  auto multiply = [&](int i, int f) {
    if constexpr (KIND == KIND_FP8) {
      part[f & 1] = mfma_step<KIND>(w[f], x[i & 1], f32x4{0.f, 0.f, 0.f, 0.f});
    } else if constexpr (KIND == KIND_FP8_WIDE) {          // (a step's weights are widened once, a row fragment before its first use)
      if (i == 0) ww[f] = widen(w[f]);
      if (f == 0) xw = widen(x[i & 1]);
      part[f & 1] = mfma_wide(ww[f], xw);
    } else acc[i][f] = mfma_step<KIND>(w[f], x[i & 1], acc[i][f]);
  };
  auto promote = [&](int i, int f) {
    if constexpr (scaled(KIND)) {
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[i][f][q] = fmaf(part[f & 1][q], s[i & 1], acc[i][f][q]);
    }
  };
  // the FMAs so far stay in front of the next branch (they would move behind it, and every partial result live until there)
  auto pin = [&] {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int f = 0; f < TN; ++f) asm volatile("" : "+v"(acc[i][f]));
  };
  // K step kb: its weight fragments, scales and first row fragment are in registers.  Every MFMA is followed by the FMAs of the one
  // before the last, also over the end of a step: a result is 11 wait states old when it is read, so the matrix pipe takes one MFMA
  // after the other with the FMAs, reads and fills in its shadow (a fragment's four MFMAs followed by its FMAs: 157 clocks for 128).
  // Row fragments are read one ahead; when the last one is, the stage is free: one barrier (which also says that stage kb + 1 has
  // landed), the fill of step kb + S, and the reads of step kb + 1's first fragments, each behind its registers' last use.  The last S
  // steps fill nothing.  A step is two halves, head and tail, split at that barrier, and the loop turns there: every read and its use
  // are in one block, so the waits count reads instead of draining them.  (No branch inside a half: the FMAs would move behind it.)
  // With two stages the weights' part of the fill goes first, behind a barrier of its own when every wave's first four MFMAs have the
  // step's weight fragments in registers: it has 1.7 steps to land instead of one (8192^3: 465 -> 449 us).
  constexpr bool W_FIRST = S == 2 && TM > 2;
  enum { STEADY, FILL_PART, DRAIN, LAST };
  int cur = 0, nxt = STAGE % (S * STAGE);                  // LDS offsets of the stages of steps kb and kb + 1
  auto slot = [&](int i, int f) {
    promote((i * TN + f + (TM - 1) * TN + 2) / TN % TM, (f + 2) % TN);          // number n - 2, or the step before's last two
    if (f == TN - 3) s[i & 1] = sx[i & 1] * sw;            // (from here on: number n - 2 is this fragment's first in the next turn)
    multiply(i, f);
  };
  // (idle: a wave all of whose outputs lie behind the last row or column only fills, and meets the others at their barriers)
  auto head = [&](int kb, auto place, auto idle) __attribute__((always_inline)) {       // MFMAs 0 .. (TM - 2) * TN + TN / 2 - 1
    constexpr int P = decltype(place)::value;
    if constexpr (decltype(idle)::value) {
      if (W_FIRST && (P == STEADY || P == FILL_PART)) {
        asm volatile("s_barrier" ::: "memory");
        fill_w(kb + S, cur, std::integral_constant<bool, P == FILL_PART>{});
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < TM - 1; ++i) {
      read_x(cur, i + 1, (i + 1) & 1);
#pragma unroll
      for (int f = 0; f < (i < TM - 2 ? TN : TN / 2); ++f) {
        if (W_FIRST && (P == STEADY || P == FILL_PART) && i == 1 && f == 0) {
          asm volatile("s_barrier" ::: "memory");
          fill_w(kb + S, cur, std::integral_constant<bool, P == FILL_PART>{});
        }
        slot(i, f);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto tail = [&](int kb, auto place, auto idle) __attribute__((always_inline)) {       // the others
    constexpr int P = decltype(place)::value;
    constexpr bool IDLE = decltype(idle)::value;
    if (P == STEADY || P == FILL_PART) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * PIECES + (W_FIRST ? WI : 0)) : "memory");
      fill_x(kb + S, cur, std::integral_constant<bool, P == FILL_PART>{});
      if (!W_FIRST) fill_w(kb + S, cur, std::integral_constant<bool, P == FILL_PART>{});
    }
    if (P == DRAIN) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (!IDLE) pin();
      if (kb + 1 == whole) clear_tail(nxt);
    }
    if constexpr (!IDLE) {
#pragma unroll
      for (int i = TM - 2; i < TM; ++i) {
        if (P != LAST && i == TM - 1) read_x(nxt, 0, 0);
#pragma unroll
        for (int f = i == TM - 2 ? TN / 2 : 0; f < TN; ++f) {
          slot(i, f);
          if (P != LAST && i == TM - 1) read_w(nxt, f);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (P != LAST) sw = read_sw(nxt);
    }
    cur = nxt, nxt = nxt + STAGE == S * STAGE ? 0 : nxt + STAGE;
  };
#define DIGA_HALF(half, kb, place) half(kb, std::integral_constant<int, place>{}, idle)
  auto all_steps = [&](auto idle) __attribute__((always_inline)) {
    int kb = 0;
    if (S < whole) {                                       // the steps that fill a whole one
      DIGA_HALF(head, 0, STEADY);
      for (; kb + 1 + S < whole; ++kb) {
        DIGA_HALF(tail, kb, STEADY);
        DIGA_HALF(head, kb + 1, STEADY);
      }
      DIGA_HALF(tail, kb, STEADY);
      ++kb;
    }
    if (kb + S < p.nk) {
      DIGA_HALF(head, kb, FILL_PART);
      DIGA_HALF(tail, kb, FILL_PART);
      ++kb;
    }
    for (; kb + 1 < p.nk; ++kb) {
      DIGA_HALF(head, kb, DRAIN);
      DIGA_HALF(tail, kb, DRAIN);
    }
    DIGA_HALF(head, kb, LAST);
    DIGA_HALF(tail, kb, LAST);
  };
#undef DIGA_HALF

#pragma unroll
  for (int t = 0; t < S; ++t)
    if (t < p.nk) fill_x(t, t * STAGE, std::true_type{}), fill_w(t, t * STAGE, std::true_type{});
  if (p.nk >= S) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 1) * PIECES) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  if (whole == 0) clear_tail(0);
  if (m0 + wm * (BM / WM) >= m1 || n0 + wn * 64 >= p.N) return all_steps(std::true_type{});
#pragma unroll
  for (int f = 0; f < TN; ++f) read_w(0, f);
  read_x(0, 0, 0);
  sw = read_sw(0);
  part[0] = part[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  all_steps(std::false_type{});
  promote(TM - 1, TN - 2);
  promote(TM - 1, TN - 1);
  pin();

  // ---- a lane's two runs of 8 consecutive outputs of each of its rows
  const int n = n0 + wn * 64 + fg * 8;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t m = m0 + (wm * TM + i) * 16 + fr;
    if (m >= m1) continue;
    float v[16];
#pragma unroll
    for (int f = 0; f < TN; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[4 * f + q] = acc[i][f][q];
    if (GROUPED && p.rows) {
      const int r = p.rows[m];
      if (r < 0 || r >= p.xrows) {
#pragma unroll
        for (int q = 0; q < 16; ++q) v[q] = 0.f;
      }
    }
    store_run<8>(p.out, p.out_type, m * p.ldo + n, v, p.N - n);
    store_run<8>(p.out, p.out_type, m * p.ldo + n + 32, v + 8, p.N - n - 32);
  }
#endif
}

// Few rows, or too few tiles for the kernel above: a block's 8 waves share one tile of 8 XG rows x 16 NT weight rows and deal the K
// steps among themselves (step j * 8 + wave).  No operand is shared between waves: each keeps a ring of D steps in LDS to itself, filled
// by LDS-DMA and waited for by its own counter, and the only barriers are those of the join: the partial outputs go through LDS,
// waves 4 .. 7 into 0 .. 3, 2, 3 into 0, 1, and 1 into 0 (a fixed order).
// What bounds it is the vector-memory path of the CU: straight into registers a fragment's 16 lanes of a quarter wave touch 16 rows,
// 64 lines for 1 KB, 38 GB/s; by LDS-DMA 8 lanes share a row's 128 bytes (33 x 2048 x 8192: 14.2 -> 6.3 us, 128 x 4096 x 4096: 8.6 against
// 13.8 of the kernel above).
template <int KIND, int XG, int NT, int D, bool GROUPED>
__global__ __launch_bounds__(512, 2) void matmul_few_kernel(MatmulParams p) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int NW = 8, BM = 8 * XG, BN = 16 * NT, MT = (XG + 1) / 2, WG = 2 * NT;
  constexpr int SCALES = (2 * MT + WG) * 1024;             // in a stage: x rows, w rows, scales
  constexpr int STAGE = SCALES + (scaled(KIND) ? 512 : 0), PIECES = XG + WG + (scaled(KIND) ? 2 : 0);
  static_assert(D * NW * STAGE <= 160 * 1024 && 4 * MT * NT * 1024 <= D * NW * STAGE, "the rings fit into LDS, the join into the rings");
  static_assert(BM <= 64, "a lane loads one row's scale");
  __shared__ __attribute__((aligned(1024))) char smem[D * NW * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  int nt, e, m0, m1;
  if (!tile_of_block<BM, GROUPED>(p, GROUPED ? 1 : 16, nt, e, m0, m1)) return;
  const int n0 = nt * BN;
  auto source_row = [&](int row) -> int64_t {              // left row behind row `row` of the tile
    int64_t m = std::min(m0 + row, m1 - 1);
    if (GROUPED && p.rows) {
      m = p.rows[m];
      if (m < 0 || m >= p.xrows) m = 0;
    }
    return m;
  };
  // fragment f's row 4 g + i is weight row 4 NT g + 4 f + i: a lane ends with 4 NT consecutive outputs
  auto swz = [](int row) { return NT == 1 ? row & 7 : (row & 3) | ((row >> 3) & 1) << 2; };
  const int64_t xfirst = GROUPED && p.rows ? 0 : m0;
  const buffer_t xtile = make_buffer(p.x + xfirst * p.ldx);
  const buffer_t wtile = make_buffer(p.w + (int64_t)e * p.wstride + (int64_t)n0 * p.ldw);
  uint32_t xoff[XG], woff[WG];
  const int row0 = lane >> 3, xchunk = ((lane & 7) ^ row0) * 16;
#pragma unroll
  for (int g = 0; g < XG; ++g) xoff[g] = (uint32_t)((source_row(8 * g + row0) - xfirst) * p.ldx);
#pragma unroll
  for (int g = 0; g < WG; ++g) woff[g] = (uint32_t)(std::min(8 * g + row0, p.N - 1 - n0) * p.ldw);
  const float* const xs = scaled(KIND) ? p.xs + source_row(lane) * p.xs_m : nullptr;       // (lanes >= BM: not used)
  const float* const ws = scaled(KIND) ? p.ws + ((int64_t)e * ((p.N + 127) >> 7) + (n0 >> 7)) * p.nk : nullptr;
  const int whole = p.Kb >> 7;
  char* const ring = smem + wave * (D * STAGE);
  auto fill = [&](int j, int st) {
    const int kb = j * NW + wave, k0 = kb * 128;
    char* s = ring + st * STAGE;
    const bool part = kb == whole;                         // a chunk behind the row's end is read from its start
#pragma unroll
    for (int g = 0; g < XG; ++g)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xtile, (lds_ptr)(s + g * 1024), 16, xoff[g] + (part && k0 + xchunk >= p.Kb ? 0 : k0 + xchunk), 0, 0, 0);
#pragma unroll
    for (int g = 0; g < WG; ++g) {
      const int c = ((lane & 7) ^ swz(8 * g + row0)) * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wtile, (lds_ptr)(s + (2 * MT + g) * 1024), 16, woff[g] + (part && k0 + c >= p.Kb ? 0 : k0 + c), 0, 0, 0);
    }
    if constexpr (scaled(KIND)) {
      __builtin_amdgcn_global_load_lds((gbl_ptr)(xs + kb * p.xs_b), (lds_ptr)(s + SCALES), 4, 0, 0);
      __builtin_amdgcn_global_load_lds((gbl_ptr)(ws + kb), (lds_ptr)(s + SCALES + 256), 4, 0, 0);
    }
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int f = 0; f < NT; ++f) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int steps = p.nk > wave ? (p.nk - wave + NW - 1) / NW : 0;        // of this wave
#pragma unroll
  for (int t = 0; t < D; ++t)
    if (t < steps) fill(t, t);
  int st = 0;
  for (int j = 0; j < steps; ++j) {
    if (j + D <= steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * PIECES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const char* s = ring + st * STAGE;
    i32x8 w[NT], x[MT];
    float sx[MT], sw = 0.f;
#pragma unroll
    for (int f = 0; f < NT; ++f) {
      const int r = (fr >> 2) * 4 * NT + 4 * f + (fr & 3);
      const char* q = s + 2 * MT * 1024 + r * 128;
      w[f] = read_pair(q + (fg ^ swz(r)) * 16, q + ((fg + 4) ^ swz(r)) * 16);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const char* q = s + (16 * i + fr) * 128;
      x[i] = read_pair(q + (fg ^ (fr & 7)) * 16, q + ((fg + 4) ^ (fr & 7)) * 16);
      sx[i] = scaled(KIND) ? reinterpret_cast<const float*>(s + SCALES)[16 * i + fr] : 0.f;
    }
    if constexpr (scaled(KIND)) sw = reinterpret_cast<const float*>(s + SCALES)[64];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the stage has been read: it may be filled again
    if (j + D < steps) fill(j + D, st);
    if (j * NW + wave == whole) {                          // what lies behind the row's end counts as zero
      const int left = p.Kb - whole * 128 - fg * 16;
#pragma unroll
      for (int f = 0; f < NT; ++f) w[f] = keep_pair(w[f], left);
#pragma unroll
      for (int i = 0; i < MT; ++i) x[i] = keep_pair(x[i], left);
    }
    Wide ww[NT], xw;                                       // (KIND_FP8_WIDE)
    if constexpr (KIND == KIND_FP8_WIDE) {
#pragma unroll
      for (int f = 0; f < NT; ++f) ww[f] = widen(w[f]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float sc = sx[i] * sw;
      if constexpr (KIND == KIND_FP8_WIDE) xw = widen(x[i]);
#pragma unroll
      for (int f = 0; f < NT; ++f) {
        if constexpr (scaled(KIND)) {
          f32x4 part;
          if constexpr (KIND == KIND_FP8) part = mfma_step<KIND>(w[f], x[i], f32x4{0.f, 0.f, 0.f, 0.f});
          else part = mfma_wide(ww[f], xw);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][f][q] = fmaf(part[q], sc, acc[i][f][q]);
        } else {
          acc[i][f] = mfma_step<KIND>(w[f], x[i], acc[i][f]);
        }
      }
    }
    st = st + 1 == D ? 0 : st + 1;
  }
  f32x4(*join)[MT][NT][64] = reinterpret_cast<f32x4(*)[MT][NT][64]>(smem);
#pragma unroll
  for (int half = NW / 2; half >= 1; half /= 2) {
    __syncthreads();                                       // (the first: every wave is done with its ring)
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int f = 0; f < NT; ++f) join[wave - half][i][f][lane] = acc[i][f];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int f = 0; f < NT; ++f) acc[i][f] += join[wave][i][f][lane];
    }
  }
  if (wave != 0) return;
  const int n = n0 + fg * 4 * NT;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + i * 16 + fr;
    if (m >= m1 || i * 16 + fr >= BM) continue;
    bool zero = false;
    if (GROUPED && p.rows) {
      const int r = p.rows[m];
      zero = r < 0 || r >= p.xrows;
    }
    float v[4 * NT];
#pragma unroll
    for (int f = 0; f < NT; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[4 * f + q] = zero ? 0.f : acc[i][f][q];
    store_run<4 * NT>(p.out, p.out_type, m * p.ldo + n, v, p.N - n);
  }
#endif
}

template <int KIND, int BM, int BN, int WM, int WN, int S, bool GROUPED>
void launch_tile(MatmulParams p, hipStream_t s) {
  p.ntiles = cdiv(p.N, BN);
  p.mtiles_max = (int)(GROUPED ? p.M / BM + std::min<int64_t>(p.E, p.M) : (p.M + BM - 1) / BM);
  matmul_kernel<KIND, BM, BN, WM, WN, S, GROUPED><<<dim3((unsigned)((int64_t)p.mtiles_max * p.ntiles)), WM * WN * 64, 0, s>>>(p);
}

template <int KIND, int XG, int NT, int D, bool GROUPED>
void launch_few(MatmulParams p, hipStream_t s) {
  constexpr int BM = 8 * XG;
  p.ntiles = cdiv(p.N, 16 * NT);
  p.mtiles_max = (int)(GROUPED ? p.M / BM + std::min<int64_t>(p.E, p.M) : (p.M + BM - 1) / BM);
  matmul_few_kernel<KIND, XG, NT, D, GROUPED><<<dim3((unsigned)((int64_t)p.mtiles_max * p.ntiles)), 512, 0, s>>>(p);
}

// Which kernel and tile: the least expected time in us, the root of the sum of squares of three: the CUs' work, the tiles' bytes at
// 20 TB/s from L2, and the operands' bytes once at 4.9 TB/s from memory.  turns = blocks / 256 rounded up (grouped: of
// the expected number: average group / tile rows + 0.3, which picked within 1.02 of the best of all 12 over 30 sets of 8 .. 128 groups of 1
// .. 1000 rows, even and skewed; + 0.5, half a tile lost to a group, within 1.06: 8 x 200 rows, 4096 x 2048, 31 -> 24 us).
//   few rows  turns * (K steps * pieces * 0.0112 + 0.3 + 0.1 * accumulators): a CU takes one 1 KB piece in 11 ns; a step is XG + 2 NT
//             pieces and 2 of scales; grouped blocks look their rows up first, 2.5.  Measured, in us, tile rows x weight rows:
//               16 x 2048 x 8192: 16 x 16 5.2, 16 x 32 6.1, 32 x 32 7.5; 33 x 2048 x 8192: 16 x 32 6.2, 16 x 16 7.6, 32 x 32 7.5
//               64 x 4096 x 4096: 32 x 32 7.4, 32 x 64 8.4, 16 x 32 9.3, 64 x 128 13.8; 96 x 4096 x 4096: 48 x 32 7.8, 32 x 64 8.4
//               128 x 4096 x 4096: 32 x 64 8.6, 48 x 64 9.7, 64 x 128 13.8; 192 x 4096 x 4096: 48 x 64 10.6, 64 x 128 14.0
//               256 x 4096 x 4096: 64 x 64 11.8, 64 x 128 14.1; 1024 slots over 32 experts, 2048 x 2048: 64 x 64 55, 64 x 128 34
//   tiled     K steps * alone + ends in one turn (barrier, reads and MFMAs of a step one after the other), else turns * (K steps * full +
//             ends): `ends` is a block's first fill and its stores.
//             64 x 128, 4 waves, 3 stages: 0.34, 0.296, 0.4 (512 x 4096 x 4096: 15.5; 8 waves 18.9, 48 x 64 24.4)
//             128 x 128, 8 waves, 3 stages, one block on a CU: 0.47, 0.55, 1.5 (512 x 8192 x 8192: 41.4; others 43.4, 44.1, 88.9)
//             128 x 128, 4 waves, 2 stages, two on a CU: 0.53, 0.475, 1.3 (8385 x 2048 x 2048: 45.0; others 49.3, 54.7, 61.2)
//             128 x 256, 8 waves, 2 stages, one on a CU: 0.8, 0.99, 3.8 (5482 x 1000 x 2048 bf16 in 16 groups: 32.2; 37.9, 42.5, 40.9, 48.7)
//             256 x 256, 8 waves, 2 stages, one on a CU: 1.22, 1.55, 10 (8192^3: 440; others 622, 592, 503, 524)
//   fp32 outputs of 8-bit products: half the matrix rate, and the widening: few + 0.012 per K step and accumulator; tiled in the order above 0.7,
//             0.53, 0.4; 1.02, 1.05, 1.5; 1.0, 0.87, 1.7; 1.6, 1.8, 5 (picks within 1.01 of the best of 11 over 28 sizes, dense and grouped: 517 x 1001 x
//             2064: 48 x 64 9.7, 64 x 64 10.8, 64 x 128 15.4; 256 x 4096 x 4096: 64 x 64 15.2, 64 x 128 23.7; 8192^3: 128 x 128 of 4 waves 906, 128 x 256
//             912, 64 x 128 1099; the wide 256 x 256 tile would take more than 256 registers)
// (e4m3, M x N x K; a step of 16-bit operands is half the K and the same bytes and MFMA clocks.)
// A launch has fewer than 2^32 threads: tiles that would need 2^23 blocks of 512 are left out.
constexpr int64_t MAX_BLOCKS = ((int64_t)1 << 23) - 1;

thread_local int asked_tile = -1;                          // diga_matmul_use_tile

// index of the tile, -1 where none fits one launch
template <int KIND, bool GROUPED>
int choose(const MatmulParams& p) {
  constexpr bool WIDE = KIND == KIND_FP8_WIDE;
  const double groups = GROUPED ? (double)std::min<int64_t>(p.E, p.M) : 1., avg = (double)p.M / groups;
  const double once = ((double)p.xrows + groups * p.N) * p.Kb / 4.9e6;
  auto time = [&](int bm, int bn, auto work) {
    const double mt = GROUPED ? groups * std::max(1., avg / bm + 0.3) : (double)((p.M + bm - 1) / bm), blocks = mt * ((p.N + bn - 1) / bn);
    const int64_t most = (GROUPED ? p.M / bm + std::min<int64_t>(p.E, p.M) : (p.M + bm - 1) / bm) * cdiv(p.N, bn);
    if (most > MAX_BLOCKS) return HUGE_VAL;
    const double cu = work(std::ceil(blocks / 256)), l2 = blocks * ((GROUPED ? bm : std::min<double>(bm, avg)) + bn) * p.Kb / 20e6;
    return cu * cu + l2 * l2 + once * once;
  };
  auto few = [&](int xg, int nt) {
    const double block = p.nk * (xg + 2 * nt + (scaled(KIND) ? 2 : 0)) * 0.0112 + (GROUPED ? 2.8 : 0.3) + (0.1 + (WIDE ? 0.012 * p.nk : 0.)) * ((xg + 1) / 2 * nt);
    return time(8 * xg, 16 * nt, [&](double turns) { return turns * block; });
  };
  auto tiled = [&](int bm, int bn, double alone, double full, double ends) {
    return time(bm, bn, [&](double turns) { return turns == 1. ? p.nk * alone + ends : turns * (p.nk * full + ends); });
  };
  const double t[] = {few(2, 1), few(2, 2), few(4, 2), few(6, 2), few(4, 4), few(6, 4), few(8, 4),
                      WIDE ? tiled(64, 128, 0.7, 0.53, 0.4) : tiled(64, 128, 0.34, 0.296, 0.4),
                      WIDE ? tiled(128, 128, 1.02, 1.05, 1.5) : tiled(128, 128, 0.47, 0.55, 1.5),
                      WIDE ? tiled(128, 128, 1.0, 0.87, 1.7) : tiled(128, 128, 0.53, 0.475, 1.3),
                      WIDE ? tiled(128, 256, 1.6, 1.8, 5.) : tiled(128, 256, 0.8, 0.99, 3.8),
                      WIDE ? HUGE_VAL : tiled(256, 256, 1.22, 1.55, 10.)};
  static_assert(std::size(t) == DIGA_MATMUL_TILES);
  const auto least = asked_tile >= 0 ? t + asked_tile : std::min_element(std::begin(t), std::end(t));
  return *least < HUGE_VAL ? (int)(least - t) : -1;
}

template <int KIND, bool GROUPED>
int launch(const char* who, const MatmulParams& p, hipStream_t s) {
  const int tile = choose<KIND, GROUPED>(p);
  DIGA_CHECK_ARG(tile >= 0, "%s: M=%lld x N=%d has too many tiles for one launch", who, (long long)p.M, p.N);
  const int64_t size = p.out_type == DIGA_FP32 ? 4 : 2;
  DIGA_CHECK_ARG(!rows_meet(p.out, p.M, p.ldo * size, p.N * size, p.x, p.rows ? p.xrows : p.M, p.ldx, p.Kb), "%s: the output lies on the left rows", who);
  DIGA_CHECK_ARG(!(p.E == 1 ? rows_meet(p.out, p.M, p.ldo * size, p.N * size, p.w, p.N, p.ldw, p.Kb)
                            : rows_meet(p.out, p.M, p.ldo * size, p.N * size, p.w, p.E, p.wstride, (p.N - 1) * p.ldw + p.Kb)),
                 "%s: the output lies on the weights", who);
  switch (tile) {
    case 0: launch_few<KIND, 2, 1, 2, GROUPED>(p, s); break;
    case 1: launch_few<KIND, 2, 2, 2, GROUPED>(p, s); break;
    case 2: launch_few<KIND, 4, 2, 2, GROUPED>(p, s); break;
    case 3: launch_few<KIND, 6, 2, 1, GROUPED>(p, s); break;
    case 4: launch_few<KIND, 4, 4, 1, GROUPED>(p, s); break;
    case 5: launch_few<KIND, 6, 4, 1, GROUPED>(p, s); break;
    case 6: launch_few<KIND, 8, 4, 1, GROUPED>(p, s); break;
    case 7: launch_tile<KIND, 64, 128, 2, 2, 3, GROUPED>(p, s); break;
    case 8: launch_tile<KIND, 128, 128, 4, 2, 3, GROUPED>(p, s); break;
    case 9: launch_tile<KIND, 128, 128, 2, 2, 2, GROUPED>(p, s); break;
    case 10: launch_tile<KIND, 128, 256, 2, 4, 2, GROUPED>(p, s); break;
    default:                                               // (its wide form would take more than 256 registers)
      if constexpr (KIND != KIND_FP8_WIDE) launch_tile<KIND, 256, 256, 2, 4, 2, GROUPED>(p, s);
      break;
  }
  DIGA_CHECK_LAUNCH(who);
  return DIGA_OK;
}

constexpr int64_t MAX_M = ((int64_t)1 << 31) - 1024;
constexpr int MAX_N = 1 << 24;
constexpr int MAX_GROUPS = 4096;                           // every block reads all offsets, 64 at a time
constexpr int MAX_ROW = 1 << 23;                           // bytes of an operand row: 256 of them inside a 32-bit offset

int check_product(const char* who, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* out, int out_type, int64_t ldo,
                  int64_t M, int N, int K, int size) {
  DIGA_CHECK_ARG(M >= 0 && M <= MAX_M, "%s: M=%lld rows (0 .. 2^31 - 1024)", who, (long long)M);
  DIGA_CHECK_ARG(N >= 1 && N <= MAX_N && K >= 1 && K <= MAX_ROW / size, "%s: N=%d (1 .. 2^24), K=%d (1 .. 8 MiB of a row)", who, N, K);
  DIGA_CHECK_ARG(out_type == DIGA_BF16 || out_type == DIGA_FP16 || out_type == DIGA_FP32, "%s: unknown output type %d", who, out_type);
  DIGA_CHECK_ARG(M == 0 || (x && w && out), "%s: null pointer", who);
  DIGA_CHECK_ARG(((uintptr_t)x & 15) == 0 && ((uintptr_t)w & 15) == 0 && ldx * size % 16 == 0 && ldw * size % 16 == 0,
                 "%s: operand rows must start at multiples of 16 bytes (row strides %lld, %lld elements)", who, (long long)ldx, (long long)ldw);
  DIGA_CHECK_ARG(ldw * size <= MAX_ROW && ldw >= 0 && ldx >= 0 && (M <= 1 || ldx * size <= MAX_ROW), "%s: row strides (%lld, %lld elements) above 8 MiB", who, (long long)ldx, (long long)ldw);
  const int64_t need = ((int64_t)K * size + 15) / 16 * 16 / size;
  DIGA_CHECK_ARG(ldw >= need && (M <= 1 || ldx >= need), "%s: row strides (%lld, %lld) below K=%d rounded up to 16 bytes", who, (long long)ldx, (long long)ldw, K);
  DIGA_CHECK_ARG(M <= 1 || ldo >= N, "%s: output row stride %lld below N=%d", who, (long long)ldo, N);
  return DIGA_OK;
}

int check_fp8_out(const char* who, int out_type) {
  DIGA_CHECK_ARG(out_type != DIGA_FP32, "%s: outputs are bf16 or fp16 (the e4m3 matrix pipe does not sum them to 32 bits: %s_f32 does)", who, who);
  return DIGA_OK;
}

}  // namespace

template <int KIND>
static int dense_fp8(const char* who, const void* x, int64_t ldx, const float* x_scale, int64_t x_scale_stride_m, int64_t x_scale_stride_b,
                     const void* w, int64_t ldw, const float* w_scale, void* out, int out_type, int64_t ldo, int64_t M, int N, int K, void* stream) {
  if (int rc = check_product(who, x, ldx, w, ldw, out, out_type, ldo, M, N, K, 1)) return rc;
  if (M == 0) return DIGA_OK;
  DIGA_CHECK_ARG(x_scale && w_scale, "%s: null pointer", who);
  MatmulParams p{};
  p.x = (const char*)x, p.w = (const char*)w, p.xs = x_scale, p.ws = w_scale, p.out = out;
  p.ldx = ldx, p.ldw = ldw, p.xs_m = x_scale_stride_m, p.xs_b = x_scale_stride_b, p.ldo = ldo;
  p.M = M, p.xrows = M, p.N = N, p.Kb = K, p.nk = cdiv(K, 128), p.E = 1, p.out_type = out_type;
  return launch<KIND, false>(who, p, static_cast<hipStream_t>(stream));
}

extern "C" int diga_matmul_fp8(const void* x, int64_t ldx, const float* x_scale, int64_t x_scale_stride_m, int64_t x_scale_stride_b,
                               const void* w, int64_t ldw, const float* w_scale, void* out, int out_type, int64_t ldo, int64_t M, int N,
                               int K, void* stream) {
  if (int rc = check_fp8_out("diga_matmul_fp8", out_type)) return rc;
  return dense_fp8<KIND_FP8>("diga_matmul_fp8", x, ldx, x_scale, x_scale_stride_m, x_scale_stride_b, w, ldw, w_scale, out, out_type, ldo, M, N, K, stream);
}

extern "C" int diga_matmul_fp8_f32(const void* x, int64_t ldx, const float* x_scale, int64_t x_scale_stride_m, int64_t x_scale_stride_b,
                                   const void* w, int64_t ldw, const float* w_scale, float* out, int64_t ldo, int64_t M, int N, int K, void* stream) {
  return dense_fp8<KIND_FP8_WIDE>("diga_matmul_fp8_f32", x, ldx, x_scale, x_scale_stride_m, x_scale_stride_b, w, ldw, w_scale, out, DIGA_FP32, ldo, M, N, K, stream);
}

static int check_groups(const char* who, const int32_t* offsets, int groups, const int32_t* rows, int64_t x_rows, int64_t T, int64_t ldx_bytes, int64_t row_bytes, int64_t ldw, int64_t w_stride, int N) {
  DIGA_CHECK_ARG(groups >= 1 && groups <= MAX_GROUPS, "%s: %d groups (1 .. 4096)", who, groups);
  DIGA_CHECK_ARG(x_rows >= 0 && x_rows <= MAX_M, "%s: %lld left rows", who, (long long)x_rows);
  DIGA_CHECK_ARG(T == 0 || offsets, "%s: null pointer", who);
  DIGA_CHECK_ARG(rows ? (T == 0 || x_rows > 0) : x_rows >= T, "%s: %lld left rows for %lld output rows", who, (long long)x_rows, (long long)T);
  DIGA_CHECK_ARG(!rows || x_rows <= 1 || ldx_bytes >= row_bytes, "%s: gathered rows of %lld bytes lie %lld bytes apart", who, (long long)row_bytes, (long long)ldx_bytes);
  DIGA_CHECK_ARG(!rows || (ldx_bytes <= 0xffffffffll && x_rows * ldx_bytes <= 0xffffffffll), "%s: rows are gathered from at most 4 GiB (%lld rows of %lld bytes)", who, (long long)x_rows, (long long)ldx_bytes);
  DIGA_CHECK_ARG(groups == 1 || w_stride >= (int64_t)(N - 1) * ldw, "%s: weight matrices overlap", who);
  return DIGA_OK;
}

template <int KIND>
static int grouped_fp8(const char* who, const void* x, int64_t ldx, int64_t x_rows, const float* x_scale, int64_t x_scale_stride_m, int64_t x_scale_stride_b,
                       const int32_t* rows, const void* w, int64_t ldw, int64_t w_stride, const float* w_scale, const int32_t* offsets, int groups,
                       void* out, int out_type, int64_t ldo, int64_t T, int N, int K, void* stream) {
  if (int rc = check_product(who, x, ldx, w, ldw, out, out_type, ldo, T, N, K, 1)) return rc;
  if (int rc = check_groups(who, offsets, groups, rows, x_rows, T, ldx, (K + 15) / 16 * 16, ldw, w_stride, N)) return rc;
  DIGA_CHECK_ARG(w_stride % 16 == 0, "%s: weight matrices must start at multiples of 16 bytes", who);
  if (T == 0) return DIGA_OK;
  DIGA_CHECK_ARG(x_scale && w_scale, "%s: null pointer", who);
  MatmulParams p{};
  p.x = (const char*)x, p.w = (const char*)w, p.xs = x_scale, p.ws = w_scale, p.rows = rows, p.offsets = offsets, p.out = out;
  p.ldx = ldx, p.ldw = ldw, p.wstride = w_stride, p.xs_m = x_scale_stride_m, p.xs_b = x_scale_stride_b, p.ldo = ldo;
  p.M = T, p.xrows = x_rows, p.N = N, p.Kb = K, p.nk = cdiv(K, 128), p.E = groups, p.out_type = out_type;
  return launch<KIND, true>(who, p, static_cast<hipStream_t>(stream));
}

extern "C" int diga_grouped_matmul_fp8(const void* x, int64_t ldx, int64_t x_rows, const float* x_scale, int64_t x_scale_stride_m,
                                       int64_t x_scale_stride_b, const int32_t* rows, const void* w, int64_t ldw, int64_t w_stride,
                                       const float* w_scale, const int32_t* offsets, int groups, void* out, int out_type, int64_t ldo,
                                       int64_t T, int N, int K, void* stream) {
  if (int rc = check_fp8_out("diga_grouped_matmul_fp8", out_type)) return rc;
  return grouped_fp8<KIND_FP8>("diga_grouped_matmul_fp8", x, ldx, x_rows, x_scale, x_scale_stride_m, x_scale_stride_b, rows, w, ldw, w_stride, w_scale,
                               offsets, groups, out, out_type, ldo, T, N, K, stream);
}

extern "C" int diga_grouped_matmul_fp8_f32(const void* x, int64_t ldx, int64_t x_rows, const float* x_scale, int64_t x_scale_stride_m,
                                           int64_t x_scale_stride_b, const int32_t* rows, const void* w, int64_t ldw, int64_t w_stride,
                                           const float* w_scale, const int32_t* offsets, int groups, float* out, int64_t ldo, int64_t T, int N,
                                           int K, void* stream) {
  return grouped_fp8<KIND_FP8_WIDE>("diga_grouped_matmul_fp8_f32", x, ldx, x_rows, x_scale, x_scale_stride_m, x_scale_stride_b, rows, w, ldw, w_stride, w_scale,
                                    offsets, groups, out, DIGA_FP32, ldo, T, N, K, stream);
}

extern "C" int diga_grouped_matmul(const void* x, int64_t ldx, int64_t x_rows, int type, const int32_t* rows, const void* w, int64_t ldw,
                                   int64_t w_stride, const int32_t* offsets, int groups, void* out, int out_type, int64_t ldo, int64_t T,
                                   int N, int K, void* stream) {
  const char* who = "diga_grouped_matmul";
  DIGA_CHECK_ARG(type == DIGA_BF16 || type == DIGA_FP16, "%s: operands are bf16 or fp16, got type %d", who, type);
  if (int rc = check_product(who, x, ldx, w, ldw, out, out_type, ldo, T, N, K, 2)) return rc;
  if (int rc = check_groups(who, offsets, groups, rows, x_rows, T, 2 * ldx, (2 * (int64_t)K + 15) / 16 * 16, ldw, w_stride, N)) return rc;
  DIGA_CHECK_ARG(w_stride % 8 == 0, "%s: weight matrices must start at multiples of 16 bytes", who);
  if (T == 0) return DIGA_OK;
  MatmulParams p{};
  p.x = (const char*)x, p.w = (const char*)w, p.rows = rows, p.offsets = offsets, p.out = out;
  p.ldx = 2 * ldx, p.ldw = 2 * ldw, p.wstride = 2 * w_stride, p.ldo = ldo;
  p.M = T, p.xrows = x_rows, p.N = N, p.Kb = 2 * K, p.nk = cdiv(2 * (int64_t)K, 128), p.E = groups, p.out_type = out_type;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return type == DIGA_BF16 ? launch<KIND_BF16, true>(who, p, s) : launch<KIND_FP16, true>(who, p, s);
}

extern "C" int diga_matmul_use_tile(int tile) {
  DIGA_CHECK_ARG(tile >= -1 && tile < DIGA_MATMUL_TILES, "diga_matmul_use_tile: tile %d (-1 .. %d)", tile, DIGA_MATMUL_TILES - 1);
  asked_tile = tile;
  return DIGA_OK;
}

extern "C" int diga_matmul_tile_of(int type, int out_type, int groups, int64_t M, int64_t x_rows, int N, int K) {
  const char* who = "diga_matmul_tile_of";
  DIGA_CHECK_ARG(type == DIGA_BF16 || type == DIGA_FP16 || type == DIGA_E4M3, "%s: unknown type %d", who, type);
  DIGA_CHECK_ARG(groups >= (type == DIGA_E4M3 ? 0 : 1) && groups <= MAX_GROUPS, "%s: %d groups", who, groups);
  const int size = type == DIGA_E4M3 ? 1 : 2;
  DIGA_CHECK_ARG(M >= 1 && M <= MAX_M && x_rows >= 1 && x_rows <= MAX_M && N >= 1 && N <= MAX_N && K >= 1 && K <= MAX_ROW / size, "%s: M=%lld, %lld left rows, N=%d, K=%d", who,
                 (long long)M, (long long)x_rows, N, K);
  MatmulParams p{};
  p.M = M, p.xrows = x_rows, p.N = N, p.Kb = K * size, p.nk = cdiv(p.Kb, 128), p.E = groups ? groups : 1;
  int tile;
  if (type == DIGA_BF16) tile = choose<KIND_BF16, true>(p);
  else if (type == DIGA_FP16) tile = choose<KIND_FP16, true>(p);
  else if (out_type == DIGA_FP32) tile = groups ? choose<KIND_FP8_WIDE, true>(p) : choose<KIND_FP8_WIDE, false>(p);
  else tile = groups ? choose<KIND_FP8, true>(p) : choose<KIND_FP8, false>(p);
  DIGA_CHECK_ARG(tile >= 0, "%s: M=%lld x N=%d has too many tiles for one launch", who, (long long)M, N);
  return tile;
}
