// The gated feed-forward operator's matrix products (gated_ff.hip has the entry points and the mathematics):
//
//   kForward   h  = act(x Wg^T + bg) * (x Wu^T + bu)                       out[token][feature]
//   kGateGrad  dg = dh u act'(g), du = dh act(g), g and u recomputed        out[token][feature], twice
//   kInputGrad dx = dg Wg + du Wu                                           out[token][column]
//   kWeightGrad dWg = dg^T x, dWu = du^T x                                  out[feature][column]
//
// All are D[r][c] = sum_k R(r, k) C(c, k) with the operand whose index runs fastest in the output as R: the matrix
// instruction gives a lane four consecutive r of one c, an 8- or 16-byte store.  What differs is which of an operand's
// two indices is contiguous in memory - k ("along", staged [row][128 bytes of k]) or the other one ("across", staged
// [k][row]); 16-bit operands staged across are read with the transposing LDS read (ds_read_b64_tr_b16).
//
// A workgroup computes a BR x BC tile, its wavefronts split it WR x WC.  Per step 128 bytes of k (64 16-bit values, 32
// float32) of both operands go to one of two LDS buffers; the next step's travel in registers meanwhile, loaded through
// a buffer descriptor that returns zeros for what lies outside the matrix (ragged edges cost a compare, no branch).
// One barrier a step.
//
// What bounds it (MI355X): a step of the 256 x 256 tile is 2048 cycles of the matrix cores (64 matrix instructions of 16 cycles a
// wavefront, two wavefronts a SIMD) and about 1300 of LDS (192 KB read at 256 bytes a cycle, 64 KB staged at 128), and takes
// 3000 or so.  By the counters (profiles/blocks_kernels.txt) matrix cores are busy for 61 to 68 % of it and LDS for 40 to 44 %:
// neither is full, wavefronts wait 40 to 44 % of their time, 7 to 12 % for LDS, the rest at the barrier and for their turn at
// the matrix cores.  The 128 x 128 tile moves half as much again through LDS an operation.  8192 x 2048 x 8192 bf16: forward
// 424 us, input gradient 432, weight gradient 456 (1.21 to 1.30 PFLOP/s), gate gradient 484 (1.14); the library's plain product
// of that size 452 (1.22).  18432 x 256 x 1024 bf16, where a tile has four steps: forward 30 us, gate gradient 44 (113 MB of dh,
// dg and du; matrix cores 22 %, LDS 36 %, of it a fifth bank conflicts of the epilogue), input and weight gradient in one launch
// 49.  float32: 18432 x 256 x 1024 forward 160 us, 121 of the 151 TFLOP/s of a large product.
#pragma once
#include "block_common.h"

#include <type_traits>

namespace mz_gff {

enum Mode { kForward = 0, kGateGrad = 1, kInputGrad = 2, kWeightGrad = 3 };
constexpr int tail_units(int mode) { return mode == kInputGrad ? 2 : 1; }
enum Activation { kSilu = 0, kGelu = 1, kRelu = 2, kSigmoid = 3 };

struct Args {
  // operands: one matrix for gate and one for up where there are two, the same twice where there is one
  const void* r[2];
  const void* c[4];          // kInputGrad: dg, du and, with parts, dg_lo, du_lo; kWeightGrad: the same
  int parts;                 // 1, or 2: dg and du come as two terms, the rounded value and what rounding left
  long ldr, ldc;             // elements between rows of the matrices as they lie in memory
  long nr, nc, nk;           // extents of r (kForward / kGateGrad: features), c and k - the k that the steps take
  long nk_all;               // all k: nk .. nk_all - 1 are added element by element, at most tail_units(mode) 16-byte units of them
  void* out[4];              // kGateGrad: dg, du and, with parts, dg_lo, du_lo
  long ldo;
  const void* bias[2];
  const void* dh;            // kGateGrad: [nc][nr]
  long lddh;
  float* col_partial;        // kGateGrad, optional: [tiles of c][2][nr] sums of dg and du over the tile's tokens
  float* partial;            // kInputGrad / kWeightGrad with splits > 1: [splits][problems][nc][nr]
  long nr_pad;               // kGateGrad: columns of out, nr rounded up to whole 16-byte units, written with zeros
  int activation, splits, steps_per_split;
};

// launchers, one translation unit per element type; tile: 0 = 256 x 256 (16-bit types), 1 = 128 x 128, 2 = 64 x 64
int launch_bf16(const Args& a, int mode, int tile, hipStream_t s);
int launch_f16(const Args& a, int mode, int tile, hipStream_t s);
int launch_f32(const Args& a, int mode, int tile, hipStream_t s);
// kInputGrad and kWeightGrad in one launch, both in tiles 1 or 2
int launch_both_bf16(const Args& x, const Args& w, int tile, hipStream_t s);
int launch_both_f16(const Args& x, const Args& w, int tile, hipStream_t s);
int launch_both_f32(const Args& x, const Args& w, int tile, hipStream_t s);
// kForward of at most 16 tokens
int launch_few_bf16(const Args& a, hipStream_t s);
int launch_few_f16(const Args& a, hipStream_t s);
int launch_few_f32(const Args& a, hipStream_t s);

constexpr int tile_side(int tile) { return tile == 0 ? 256 : tile == 1 ? 128 : 64; }

}  // namespace mz_gff

#ifdef MZ_GFF_KERNELS
namespace {

using mz_gff::Args;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
template <typename T> using vec4 = T __attribute__((ext_vector_type(4)));
template <typename T> using vec8 = T __attribute__((ext_vector_type(8)));

// D += R C over the k that a lane's 16 bytes of each operand hold: 32 values of k a matrix instruction for the 16-bit
// types; float32 takes four instructions of 4, k = 4 (lane / 16) + j in the j-th - the same k for both operands, which
// is all that matters.
__device__ __forceinline__ f32x4 mma(u32x4 r, u32x4 c, f32x4 d, __bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec8<__bf16>, r), __builtin_bit_cast(vec8<__bf16>, c), d, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(u32x4 r, u32x4 c, f32x4 d, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec8<_Float16>, r), __builtin_bit_cast(vec8<_Float16>, c), d, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(u32x4 r, u32x4 c, f32x4 d, float) {
  const f32x4 a = __builtin_bit_cast(f32x4, r), b = __builtin_bit_cast(f32x4, c);
#pragma unroll
  for (int j = 0; j < 4; ++j) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], d, 0, 0, 0);
  return d;
}

// exp and reciprocal of the 16-bit types' activations: the hardware's, good to float32's last bits near zero and to
// 2^-17 relative at |x| = 80 - far below the 2^-9 / 2^-12 rounding of the result.  float32 results take the library's.
template <typename T> __device__ __forceinline__ float act_exp(float v) { return __expf(v); }
template <> __device__ __forceinline__ float act_exp<float>(float v) { return expf(v); }
template <typename T> __device__ __forceinline__ float act_rcp(float v) { return __builtin_amdgcn_rcpf(v); }
template <> __device__ __forceinline__ float act_rcp<float>(float v) { return 1.f / v; }

// The normal distribution at g from e = exp(-g^2 / 2), which the gradient needs anyway: up to -0, e t P(t) with t = 1 / (1 + 0.34 |g|)
// and P fitted by linear programming to erfcx(|g| / sqrt 2) / (2 t) over |g| <= 14 (at 14 e is below float32's range), off by 5.2 x
// 2^-24 in float32 arithmetic; above, 1 less that.  So a GELU keeps its digits at the lower end, where 1 + erf has a tenth of
// them left at -5 and none at -6 (18432 x 256 x 1024 forward, bf16: 1 + erff 40 us, erfcf 45, this 36; float32 164, 170, 165).
template <typename T> __device__ __forceinline__ float normal_cdf(float g, float e) {
  const float t = act_rcp<T>(1.f + 0.34f * fabsf(g));
  float q = -0.0253522731f;
  q = q * t + 0.135834962f;
  q = q * t - 0.265791029f;
  q = q * t + 0.194154903f;
  q = q * t - 0.0395074934f;
  q = q * t + 0.113314614f;
  q = q * t + 0.115668818f;
  q = q * t + 0.136054039f;
  q = q * t + 0.135623455f;
  q *= t * e;
  return g < 0.f ? q : 1.f - q;
}
template <typename T> __device__ __forceinline__ float bell(float g) { return act_exp<T>(-0.5f * g * g); }

template <typename T, int KIND> __device__ __forceinline__ float activate(float g) {
  if constexpr (KIND == mz_gff::kRelu) return g < 0.f ? 0.f : g;      // a NaN stays one
  if constexpr (KIND == mz_gff::kGelu) return g * normal_cdf<T>(g, bell<T>(g));
  const float sig = act_rcp<T>(1.f + act_exp<T>(-g));
  return KIND == mz_gff::kSilu ? g * sig : sig;
}
// act(g) and act'(g)
template <typename T, int KIND> __device__ __forceinline__ void activate_grad(float g, float& act, float& slope) {
  if constexpr (KIND == mz_gff::kRelu) {
    act = g < 0.f ? 0.f : g;
    slope = g > 0.f ? 1.f : 0.f;
  } else if constexpr (KIND == mz_gff::kGelu) {
    const float e = bell<T>(g), cdf = normal_cdf<T>(g, e);
    act = g * cdf;
    slope = cdf + g * e * 0.39894228040143268f;
  } else if constexpr (KIND == mz_gff::kSilu) {
    const float sig = act_rcp<T>(1.f + act_exp<T>(-g));
    act = g * sig;
    slope = sig * (1.f + g * (1.f - sig));
  } else {                                 // 1 - sigmoid(g) = sigmoid(-g), from exp(-|g|): neither loses the small one's digits
    const float e = act_exp<T>(-fabsf(g)), large = act_rcp<T>(1.f + e), small = e * large;
    act = g < 0.f ? small : large;
    slope = small * large;
  }
}
// f(integral constant of the activation): the choice is made once, outside the loops over outputs.  FIXED >= 0: it is
// that one (the kernels whose registers four copies of the epilogue in one function would cost).
constexpr int kAnyActivation = -1;
template <int FIXED, typename F> __device__ __forceinline__ void with_activation(int kind, F&& f) {
  if constexpr (FIXED != kAnyActivation) return f(std::integral_constant<int, FIXED>{});
  if (kind == mz_gff::kSilu) f(std::integral_constant<int, mz_gff::kSilu>{});
  else if (kind == mz_gff::kGelu) f(std::integral_constant<int, mz_gff::kGelu>{});
  else if (kind == mz_gff::kRelu) f(std::integral_constant<int, mz_gff::kRelu>{});
  else f(std::integral_constant<int, mz_gff::kSigmoid>{});
}

constexpr unsigned kOutside = 0x80000000u;   // a byte offset no descriptor below covers: the load returns zeros

// One operand's share of a step.  ACROSS: the matrix lies [k][row], else [row][k].  B rows a tile, NT threads.
template <typename T, bool ACROSS, int B, int NT> struct Operand {
  static constexpr int EC = 16 / (int)sizeof(T);        // elements of a 16-byte unit
  static constexpr int KS = 128 / (int)sizeof(T);       // k of a step
  static constexpr int UNITS = B * 8 / NT;              // 16-byte units a thread moves per step
  static constexpr int UPR = ACROSS ? B / EC : 8;       // units of a staged row
  static constexpr int READS = !ACROSS ? 1 : sizeof(T) == 2 ? 2 : 4;   // LDS reads of a fragment
  static_assert(B * 8 % NT == 0 && NT % UPR == 0, "whole rows per round of threads");
  static constexpr int RPR = NT / UPR;                  // staged rows a round covers
  unsigned off[UNITS];                                  // byte offset from the step's origin
  int row0, unit;                                       // staged row of the first unit; unit within the row

  // the unit of a staged row where global unit u of that row is kept, so that the 16 x 16 blocks the wavefronts read
  // fall on different banks: along - 16 rows at one unit, rows are 128 bytes and the banks 256, so pairs of rows move
  // together; across - 16-bit: rows {8 g + 0..3} (or + 4..7) of two lane groups, a block being two units; float32:
  // rows 4 g + j of four lane groups, a block being four units.
  static __device__ __forceinline__ int place(int row, int u) {
    if constexpr (!ACROSS) return u ^ ((row >> 1) & 7);
    else if constexpr (sizeof(T) == 4) return u ^ (((row >> 2) & 3) << 2);
    else return u ^ (across_swizzle(row) << 1);
  }
  static __device__ __forceinline__ int across_swizzle(int row) {
    if constexpr (B >= 128) return (row & 3) | (((row >> 3) & 1) << 2);
    else return ((row >> 1) & 1) | (((row >> 3) & 1) << 1);   // four blocks a row, two rows to 256 bytes
  }

  __device__ __forceinline__ void init(int tid, long ld, long rows_left) {
    row0 = tid / UPR;
    unit = tid % UPR;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int row = row0 + i * RPR;
      if constexpr (ACROSS) off[i] = (long)unit * EC < rows_left ? (unsigned)(row * ld * (long)sizeof(T) + unit * 16) : kOutside;
      else off[i] = row < rows_left ? (unsigned)(row * ld * (long)sizeof(T) + unit * 16) : kOutside;
    }
  }
  // unit i of the step whose origin - the matrix element of (tile row 0, k = k0) - `rs` starts at; k_left: how many of the
  // step's k exist
  __device__ __forceinline__ u32x4 load(__amdgpu_buffer_rsrc_t rs, int k_left, int i) const {
    const bool inside = ACROSS ? row0 + i * RPR < k_left : unit * EC < k_left;
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(inside ? off[i] : kOutside), 0, 0));
  }
  __device__ __forceinline__ void stage(char* lds, int i, u32x4 v) const {
    const int row = row0 + i * RPR;
    *reinterpret_cast<u32x4*>(lds + row * (UPR * 16) + place(row, unit) * 16) = v;
  }
  // lane's 16 bytes of block `blk` (rows 16 blk ..) at sub-step `sub` of the step's two
  static __device__ __forceinline__ u32x4 fragment(const char* lds, int blk, int sub, int lane) {
    const int g = lane >> 4, l = lane & 15;
    if constexpr (!ACROSS) {
      const int row = blk * 16 + l;
      return *reinterpret_cast<const u32x4*>(lds + row * 128 + (((sub * 4 + g) ^ ((row >> 1) & 7)) << 4));
    } else if constexpr (sizeof(T) == 2) {
      s16x8 out;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = sub * 32 + g * 8 + h * 4 + (l >> 2);
        const char* p = lds + row * (UPR * 16) + ((blk ^ across_swizzle(row)) << 5) + (l & 3) * 8;
        const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
#pragma unroll
        for (int j = 0; j < 4; ++j) out[h * 4 + j] = t[j];
      }
      return __builtin_bit_cast(u32x4, out);
    } else {
      u32x4 out;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = sub * 16 + g * 4 + j;
        out[j] = *reinterpret_cast<const unsigned*>(lds + row * (UPR * 16) + ((blk ^ ((row >> 2) & 3)) << 6) + l * 4);
      }
      return out;
    }
  }
};

// How many of n things fall to the i-th of `parts` turns: turn i takes [i n / parts, (i + 1) n / parts).
constexpr int turn_begin(int i, int n, int parts) { return i * n / parts; }
constexpr int turn_count(int i, int n, int parts) { return (i + 1) * n / parts - i * n / parts; }
// The order of a half step's instructions, which is the order they are written in: per 16-row block of R its matrix
// instructions, then that turn's LDS reads, LDS writes and loads.  (Left to itself the compiler moves the reads to right
// before their use and waits for each.)
template <int I, int BLOCKS, int MMAS, int R_READS, int C_BLOCKS, int C_READS, int UNITS>
__device__ __forceinline__ void half_step_order() {
  if constexpr (I < BLOCKS) {
    constexpr int units = turn_count(I, UNITS, BLOCKS);
    __builtin_amdgcn_sched_group_barrier(0x008, MMAS, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R_READS + C_READS * turn_count(I, C_BLOCKS, BLOCKS), 0);
    if constexpr (units > 0) {
      __builtin_amdgcn_sched_group_barrier(0x200, units, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, units, 0);
    }
    half_step_order<I + 1, BLOCKS, MMAS, R_READS, C_BLOCKS, C_READS, UNITS>();
  }
}

template <typename T, int MODE, int BR, int BC, int WR, int WC, int ACT>
__device__ __forceinline__ void gff_gemm(Args a, unsigned block, unsigned blocks, char* lds) {
  using namespace mz_gff;
  constexpr int NT = WR * WC * 64;
  constexpr bool kPair = MODE == kForward || MODE == kGateGrad;       // a tile's R rows: half gate, half up features
  constexpr bool kRAcross = !kPair, kCAcross = MODE == kWeightGrad;
  using OpR = Operand<T, kRAcross, BR, NT>;
  using OpC = Operand<T, kCAcross, BC, NT>;
  constexpr int KS = OpR::KS;
  constexpr int RM = BR / WR / 16, CN = BC / WC / 16;                 // 16 x 16 blocks of a wavefront
  constexpr int TR = kPair ? BR / 2 : BR;                             // output rows (r) of a tile
  // lds: two buffers of (BR + BC) x 128 bytes, then biases
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave / WC, wc = wave % WC;

  // ---- this workgroup's tiles.  Workgroups go to the 8 XCDs in turn: XCD x takes the x-th run of consecutive tiles, and
  // consecutive tiles walk 8 tiles of c under each tile of r, so that an L2 holds what its workgroups share.  A pair
  // product's workgroups stay for several tiles - the next one's first units are on their way while a tile's epilogue runs -
  // the plain products' take one each.
  const unsigned tiles_r = (unsigned)((a.nr + TR - 1) / TR), tiles_c = (unsigned)((a.nc + BC - 1) / BC);
  const unsigned problems = MODE == kWeightGrad ? 2 : 1;
  const unsigned per_problem = tiles_r * tiles_c, total = per_problem * problems * (unsigned)a.splits;
  const unsigned per_xcd = (total + 7) / 8;
  const unsigned xcd0 = (block & 7) * per_xcd;                        // the XCD's first tile
  unsigned local = block >> 3;                                        // of its run
  if (local >= per_xcd || xcd0 + local >= total) return;
  long r0 = 0, c0 = 0;
  int which = 0, split = 0;
  constexpr unsigned kGroup = 8;
  auto locate = [&]() __attribute__((always_inline)) {
    const unsigned id = xcd0 + local, job = id / per_problem, t = id - job * per_problem;
    which = MODE == kWeightGrad ? (int)(job % 2) : 0;
    split = (int)(MODE == kWeightGrad ? job / 2 : job);
    const unsigned band = t / (kGroup * tiles_r), in_band = t - band * (kGroup * tiles_r);
    const unsigned band_c = tiles_c - band * kGroup < kGroup ? tiles_c - band * kGroup : kGroup;
    r0 = (long)(in_band / band_c) * TR;
    c0 = (long)(band * kGroup + in_band % band_c) * BC;
  };
  locate();

  // ---- operands
  OpR opr;
  OpC opc;
  // a pair tile's two halves are two matrices: the rounds of threads split evenly between them
  constexpr int kHalf = kPair ? OpR::UNITS / 2 : OpR::UNITS;
  static_assert(!kPair || (OpR::UNITS % 2 == 0 && kHalf * OpR::RPR == BR / 2), "rounds cover a half");
  auto aim = [&]() __attribute__((always_inline)) {
    opr.init(tid, a.ldr, a.nr - r0);
    if constexpr (kPair) {        // rows of the second half are rows 0 .. BR/2 of the other matrix
#pragma unroll
      for (int i = 0; i < kHalf; ++i) opr.off[kHalf + i] = opr.off[i];
    }
    opc.init(tid, a.ldc, a.nc - c0);
  };
  aim();
  // steps: kInputGrad runs over the features of dg and then over those of du; where these come in two parts - small
  // problems, in the smallest tiles - the second parts' steps follow the first's
  constexpr int kParts = BR == 64 && sizeof(T) == 2 && !kPair ? 2 : 1, kSides = MODE == kInputGrad ? 2 : 1, kSegs = kParts * kSides;
  const long seg_steps = (a.nk + KS - 1) / KS;
  const int segs = kSides * (kParts == 2 ? a.parts : 1);
  const long all_steps = seg_steps * segs;
  auto c_matrix = [&](int seg) __attribute__((always_inline)) {
    const int i = MODE == kInputGrad ? seg : which + 2 * seg;
    const void* m = i == 0 ? a.c[0] : a.c[1];
    if constexpr (kParts == 2) m = i < 2 ? m : i == 2 ? a.c[2] : a.c[3];
    return static_cast<const T*>(m);
  };
  const long first = (long)split * a.steps_per_split;
  const long last = first + a.steps_per_split < all_steps ? first + a.steps_per_split : all_steps;

  // a step's units, R's and then C's, travel in v; unit u of step s is loaded from source(s) and staged in a buffer
  constexpr int kUnits = OpR::UNITS + OpC::UNITS;
  u32x4 v[kUnits];
  struct Source {
    __amdgpu_buffer_rsrc_t r[2], c;
    int k_left;
  };
  auto source = [&](long s) __attribute__((always_inline)) {
    int seg = 0;
#pragma unroll
    for (int i = 1; i < kSegs; ++i) seg += i < segs && s >= i * seg_steps ? 1 : 0;   // past the end: in the last, behind its k
    const long k0 = (s - seg * seg_steps) * KS, left = a.nk - k0;
    const T* cm = c_matrix(seg);
    const T* rm0 = static_cast<const T*>(MODE == kInputGrad && (seg & 1) ? a.r[1] : a.r[0]);
    const T* rm1 = kPair ? static_cast<const T*>(a.r[1]) : rm0;
    const long ro = kPair ? r0 * a.ldr + k0 : k0 * a.ldr + r0, co = kCAcross ? k0 * a.ldc + c0 : c0 * a.ldc + k0;
    Source src;
    src.r[0] = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(rm0) + ro, 0, 0x7fffffff, 0x00020000);
    src.r[1] = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(rm1) + ro, 0, 0x7fffffff, 0x00020000);
    src.c = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(cm) + co, 0, 0x7fffffff, 0x00020000);
    src.k_left = left < 0 ? 0 : left < KS ? (int)left : KS;
    return src;
  };
  auto load_unit = [&](const Source& src, int u) __attribute__((always_inline)) {
    if (u < OpR::UNITS) v[u] = opr.load(src.r[kPair && u >= kHalf ? 1 : 0], src.k_left, u);
    else v[u] = opc.load(src.c, src.k_left, u - OpR::UNITS);
  };
  auto stage_unit = [&](int buf, int u) __attribute__((always_inline)) {
    char* base = lds + buf * ((BR + BC) * 128);
    if (u < OpR::UNITS) opr.stage(base, u, v[u]);
    else opc.stage(base + BR * 128, u - OpR::UNITS, v[u]);
  };

  f32x4 acc[RM][CN];
  // the tile's 16-row block that this wavefront's block i is (pair tiles: the same features of both halves)
  auto r_block = [&](int i) {
    if constexpr (kPair) return (i / (RM / 2)) * (BR / 32) + wr * (RM / 2) + i % (RM / 2);
    else return wr * RM + i;
  };

  // A step has two halves, 64 bytes of k each, whose operands are in registers when they begin: while the first half's
  // matrix instructions run, the second half's operands are read from LDS, the next step's units (loaded a step ago) are
  // staged in the other buffer and the ones after that are sent for; then the barrier; while the second half runs, the
  // next step's first operands are read.  No branch in the loop: steps past the end load nothing (every offset is
  // outside) and stage zeros.
  constexpr int kMmas = sizeof(T) == 4 ? 4 : 1;
  u32x4 rf[RM], cf[2][CN];
  // the next tile's first units are loaded before this one's epilogue where the registers have room for them
  constexpr bool kAhead = kPair && BR != 256;
  auto start_tile = [&]() __attribute__((always_inline)) {
    const Source src = source(first);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) load_unit(src, u);
  };
  // the tile's biases, as float32 behind the two buffers: [gate, up][TR]
  auto load_bias = [&]() __attribute__((always_inline)) {
    float* bias = reinterpret_cast<float*>(lds + 2 * (BR + BC) * 128);
    for (int i = tid; i < 2 * TR; i += NT) {
      const T* b = static_cast<const T*>(a.bias[i / TR]);
      const long f = r0 + i % TR;
      bias[i] = b && f < a.nr ? (float)b[f] : 0.f;
    }
  };
  // of the lane's four features in the wavefront's block i
  constexpr bool kBiasFirst = kPair && sizeof(T) == 2;
  constexpr long kBiasFirstK = 1 << 15;
  const int lr = (lane >> 4) * 4, lc = lane & 15;
  auto bias_of = [&](int i) __attribute__((always_inline)) {
    const int f = (i / (RM / 2)) * TR + (wr * (RM / 2) + i % (RM / 2)) * 16 + lr;
    return *reinterpret_cast<const f32x4*>(lds + 2 * (BR + BC) * 128 + f * 4);
  };
  // The epilogue is each wavefront's own: it goes over its part of the tile - WF features (columns) of CN 16-token blocks - in
  // passes of PR tokens that go through a region of LDS no other wavefront touches, so that memory is read and written in whole
  // 16-byte units of consecutive features, whatever the rows' alignment, and no wavefront waits for another.
  constexpr int WF = TR / WR, EU = WF / OpR::EC;                       // features; 16-byte units of them
  constexpr int PR = 16 * EU < 64 ? 64 / EU : 16, PU = PR * EU / 64;   // tokens of a pass; units a lane moves in one
  constexpr int PASSES = CN * 16 / PR;
  static_assert(CN * 16 % PR == 0 && PR * EU % 64 == 0, "whole passes");
  // what the wavefront has written to LDS before, it may read in other lanes after
  auto wave_sync = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  // the last step has nothing to stage or to read ahead
  auto step = [&](const char* here, const char* next, int next_buf, long s, auto is_last) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(is_last)::value;
    Source after;
    if constexpr (!LAST) after = source(s + 2);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
      for (int j = 0; j < CN; ++j) acc[i][j] = mma(rf[i], cf[0][j], acc[i][j], T{});
#pragma unroll
      for (int j = turn_begin(i, CN, RM); j < turn_begin(i + 1, CN, RM); ++j)
        cf[1][j] = OpC::fragment(here + BR * 128, wc * CN + j, 1, lane);
      rf[i] = OpR::fragment(here, r_block(i), 1, lane);
      if constexpr (!LAST) {
#pragma unroll
        for (int u = turn_begin(i, kUnits, RM); u < turn_begin(i + 1, kUnits, RM); ++u) {
          stage_unit(next_buf, u);
          load_unit(after, u);
        }
      }
    }
    half_step_order<0, RM, CN * kMmas, OpR::READS, CN, OpC::READS, LAST ? 0 : kUnits>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
      for (int j = 0; j < CN; ++j) acc[i][j] = mma(rf[i], cf[1][j], acc[i][j], T{});
      if constexpr (!LAST) {
#pragma unroll
        for (int j = turn_begin(i, CN, RM); j < turn_begin(i + 1, CN, RM); ++j)
          cf[0][j] = OpC::fragment(next + BR * 128, wc * CN + j, 0, lane);
        rf[i] = OpR::fragment(next, r_block(i), 0, lane);
      }
    }
    if constexpr (!LAST) half_step_order<0, RM, CN * kMmas, OpR::READS, CN, OpC::READS, 0>();
  };
  start_tile();
  for (;;) {
    if constexpr (kPair) load_bias();
    const Source second = source(first + 1);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      stage_unit(0, u);
      load_unit(second, u);
    }
    __syncthreads();
    // a pair product's sums start at the biases in the 16-bit types: two additions less for every output of the epilogue, 1.9 us
    // of the 18432 x 256 x 1024 bf16 forward pass.  Each of the sum's additions, one for 32 values of k, then loses up to 2^-24
    // of the bias: 2^-14 of it at K = 2^15, an eighth of float16's half step, so that longer sums add it last, and so does
    // float32, which keeps those digits.
    const bool bias_now = kBiasFirst && a.nk_all <= kBiasFirstK;
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const f32x4 start = bias_now ? bias_of(i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < CN; ++j) acc[i][j] = start;
    }
#pragma unroll
    for (int j = 0; j < CN; ++j) cf[0][j] = OpC::fragment(lds + BR * 128, wc * CN + j, 0, lane);
#pragma unroll
    for (int i = 0; i < RM; ++i) rf[i] = OpR::fragment(lds, r_block(i), 0, lane);
    int buf = 0;
    for (long s = first; s + 1 < last; ++s, buf ^= 1)
      step(lds + buf * ((BR + BC) * 128), lds + (buf ^ 1) * ((BR + BC) * 128), buf ^ 1, s, std::false_type{});
    // kGateGrad: the wavefront's part of dh, sent for as a whole (up to 32 registers) before the last step, which loads nothing
    // else, or, in float32's larger tile, two passes ahead; a tile with a ragged edge reads its dh pass by pass
    constexpr int kDhPasses = sizeof(T) == 2 || BR == 64 ? PASSES : 2;
    const bool full = r0 + TR <= a.nr && c0 + BC <= a.nc;
    Vec16<T> dh_unit[MODE == kGateGrad ? kDhPasses : 1][PU];
    const T* const dh = MODE == kGateGrad ? static_cast<const T*>(a.dh) + (c0 + wc * CN * 16) * a.lddh + r0 + wr * WF : nullptr;
    auto load_dh = [&](int p) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < PU; ++n) {
        const int e = lane + n * 64;
        dh_unit[p % kDhPasses][n].load(dh + (p * PR + e / EU) * a.lddh + e % EU * OpR::EC);
      }
    };
    if (MODE == kGateGrad && full) {
#pragma unroll
      for (int p = 0; p < kDhPasses; ++p) load_dh(MODE == kGateGrad ? p : 0);
    }
    if (first < last) step(lds + buf * ((BR + BC) * 128), nullptr, 0, last - 1, std::true_type{});
    __syncthreads();               // the epilogue uses the buffers
    __builtin_amdgcn_sched_barrier(0);                                  // and none of its registers before

    // ---- the k left out of the steps: staged as rows of one unit (kInputGrad: two) for each of dg, du and their second
    // parts, one or two more half steps
    if (a.nk_all > a.nk && split == a.splits - 1) {
      using TailR = Operand<T, false, BR, NT>;
      using TailC = Operand<T, false, BC, NT>;
      constexpr int kTail = tail_units(MODE);
      for (int row = tid; row < BR + BC; row += NT) {
        const bool is_r = row < BR;
        const int q = is_r ? row : row - BR;
        char* base = lds + (is_r ? 0 : BR * 128) + q * 128;
#pragma unroll
        for (int unit = 0; unit < (kSegs * kTail > 4 ? 8 : 4); ++unit) {
          const int seg = unit / kTail;
          const long k = a.nk + unit % kTail * OpR::EC;
          Vec16<T> e;
#pragma unroll
          for (int t = 0; t < OpR::EC; ++t) e.v[t] = (T)0.f;
          if (seg < kSegs && (seg < kSides || a.parts == 2)) {
            const T* p;
            long along;              // elements between k's
            bool exists;
            if (is_r) {
              const int r = kPair ? q % TR : q;
              exists = r0 + r < a.nr;
              p = static_cast<const T*>((kPair ? q / TR : MODE == kInputGrad ? seg & 1 : 0) ? a.r[1] : a.r[0]) +
                  (kRAcross ? k * a.ldr + r0 + r : (r0 + r) * a.ldr + k);
              along = kRAcross ? a.ldr : 1;
            } else {
              exists = c0 + q < a.nc;
              p = c_matrix(seg) + (kCAcross ? k * a.ldc + c0 + q : (c0 + q) * a.ldc + k);
              along = kCAcross ? a.ldc : 1;
            }
#pragma unroll
            for (int t = 0; t < OpR::EC; ++t)
              if (exists && k + t < a.nk_all) e.v[t] = p[t * along];
          }
          e.store(reinterpret_cast<T*>(base + TailR::place(q, unit) * 16));
        }
      }
      __syncthreads();
#pragma unroll
      for (int sub = 0; sub < (kSegs * kTail > 4 ? 2 : 1); ++sub) {
#pragma unroll
        for (int j = 0; j < CN; ++j) cf[0][j] = TailC::fragment(lds + BR * 128, wc * CN + j, sub, lane);
#pragma unroll
        for (int i = 0; i < RM; ++i) {
          rf[i] = TailR::fragment(lds, r_block(i), sub, lane);
#pragma unroll
          for (int j = 0; j < CN; ++j) acc[i][j] = mma(rf[i], cf[0][j], acc[i][j], T{});
        }
      }
      __syncthreads();
    }

    if (kBiasFirst && !bias_now) {
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < CN; ++j) acc[i][j] += bias_of(i);
    }

    const long er = r0, ec = c0;     // the tile whose epilogue follows
    bool more = false;
    if constexpr (kAhead) {
      local += blocks >> 3;
      more = local < per_xcd && xcd0 + local < total;
      if (more) {
        locate();
        aim();
        if constexpr (kAhead) start_tile();
      }
    }

    // ---- epilogue: lane holds r = 16 block + 4 (lane / 16) + 0..3 of c = 16 block + lane % 16
    if constexpr (kPair) {
      constexpr bool kLow = MODE == kGateGrad && BR == 64 && sizeof(T) == 2;      // second parts are written for small problems
      // regions of a wavefront: h; or dh and then dg in its place, du and their second parts
      constexpr int kPitch = WF * (int)sizeof(T) + 16, kRegion = PR * kPitch, kRegions = kLow ? 4 : MODE == kGateGrad ? 2 : 1;
      char* region = lds + wave * (kRegions * kRegion);
      float* colsum = reinterpret_cast<float*>(lds + WR * WC * (kRegions * kRegion));    // kGateGrad: [WC][2][TR]
      const long wf = er + wr * WF, wt = ec + wc * CN * 16;            // the wavefront's first feature, token
      const long limit = (MODE == kGateGrad ? a.nr_pad : a.nr) - wf;   // columns of the outputs from wf on
      with_activation<ACT>(a.activation, [&](auto kind) __attribute__((always_inline)) {
        constexpr int KIND = decltype(kind)::value;
        float sg[RM / 2][4], su[RM / 2][4];
#pragma unroll
        for (int i = 0; i < RM / 2; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) sg[i][q] = su[i][q] = 0.f;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          if constexpr (MODE == kGateGrad) {
            if (full) {
#pragma unroll
              for (int n = 0; n < PU; ++n) {
                const int e = lane + n * 64;
                dh_unit[p % kDhPasses][n].store(reinterpret_cast<T*>(region + e / EU * kPitch + e % EU * 16));
              }
              if (p + kDhPasses < PASSES) load_dh(p + kDhPasses);
            } else {
#pragma unroll 1
              for (int e = lane; e < PR * EU; e += 64) {
                const long c = wt + p * PR + e / EU, f = wf + e % EU * OpR::EC;
                Vec16<T> d;
                d.load_upto(static_cast<const T*>(a.dh) + c * a.lddh + f, c < a.nc ? a.nr - f : 0);
                d.store(reinterpret_cast<T*>(region + e / EU * kPitch + e % EU * 16));
              }
            }
            wave_sync();
          }
#pragma unroll
          for (int b = 0; b < PR / 16; ++b) {
            const int j = p * (PR / 16) + b;
            const bool token = wt + j * 16 + lc < a.nc;
#pragma unroll
            for (int i = 0; i < RM / 2; ++i) {
              const int fw = i * 16 + lr;                              // feature within the wavefront's
              char* at = region + (b * 16 + lc) * kPitch + fw * (int)sizeof(T);
              f32x4 g = acc[i][j], u = acc[i + RM / 2][j];
              if constexpr (!kBiasFirst) {
                g += bias_of(i);
                u += bias_of(i + RM / 2);
              }
              vec4<T> o0, o1, l0, l1;
              if constexpr (MODE == kForward) {
#pragma unroll
                for (int q = 0; q < 4; ++q) o0[q] = (T)(activate<T, KIND>(g[q]) * u[q]);
              } else {
                const vec4<T> d = *reinterpret_cast<const vec4<T>*>(at);
                float dg[4], du[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  float act, slope;
                  activate_grad<T, KIND>(g[q], act, slope);
                  dg[q] = (float)d[q] * u[q] * slope;
                  du[q] = (float)d[q] * act;
                }
                if (!full) {         // what lies past the last token or feature counts as zero
#pragma unroll
                  for (int q = 0; q < 4; ++q) {
                    const bool exists = token && wf + fw + q < a.nr;
                    dg[q] = exists ? dg[q] : 0.f;
                    du[q] = exists ? du[q] : 0.f;
                  }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  sg[i][q] += dg[q];
                  su[i][q] += du[q];
                  o0[q] = (T)dg[q];
                  o1[q] = (T)du[q];
                  if constexpr (kLow) {
                    l0[q] = (T)(dg[q] - (float)o0[q]);
                    l1[q] = (T)(du[q] - (float)o1[q]);
                  }
                }
                *reinterpret_cast<vec4<T>*>(at + kRegion) = o1;
                if constexpr (kLow) {
                  if (a.parts == 2) {
                    *reinterpret_cast<vec4<T>*>(at + 2 * kRegion) = l0;
                    *reinterpret_cast<vec4<T>*>(at + 3 * kRegion) = l1;
                  }
                }
              }
              *reinterpret_cast<vec4<T>*>(at) = o0;
            }
          }
          wave_sync();
#pragma unroll
          for (int n = 0; n < PU; ++n) {
            const int e = lane + n * 64, f = e % EU * OpR::EC;
            const long c = wt + p * PR + e / EU, left = limit - f;
            if (c >= a.nc || left <= 0) continue;
#pragma unroll
            for (int w = 0; w < kRegions; ++w) {
              if (w >= 2 && a.parts != 2) break;
              Vec16<T> o;
              o.load(reinterpret_cast<const T*>(region + w * kRegion + e / EU * kPitch + e % EU * 16));
              o.store_upto(static_cast<T*>(a.out[w]) + c * a.ldo + wf + f, left);
            }
          }
          wave_sync();
        }
        if constexpr (MODE == kGateGrad) {
          if (a.col_partial) {       // over the 16 tokens of the lanes, then (below) over the wavefronts side by side
#pragma unroll
            for (int i = 0; i < RM / 2; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int fr = (wr * (RM / 2) + i) * 16 + lr + q;
                const float g = lanes_sum<16>(sg[i][q]), u = lanes_sum<16>(su[i][q]);
                if (lc == 0) {
                  colsum[(wc * 2 + 0) * TR + fr] = g;
                  colsum[(wc * 2 + 1) * TR + fr] = u;
                }
              }
            __syncthreads();
            for (int i = tid; i < 2 * TR; i += NT) {
              const int side = i / TR, f = i % TR;
              if (er + f >= a.nr) continue;
              float v = 0.f;
#pragma unroll
              for (int w = 0; w < WC; ++w) v += colsum[(w * 2 + side) * TR + f];
              a.col_partial[((ec / BC) * 2 + side) * a.nr + er + f] = v;
            }
          }
        }
      });
    } else {
      // out in elements of O: the result itself, or float32 partial results of a cut sum
      auto finish = [&](auto* out, long ldo) __attribute__((always_inline)) {
        using O = std::remove_pointer_t<decltype(out)>;
        constexpr int EO = Vec16<O>::N, UO = WF / EO, kPitch = WF * (int)sizeof(O) + 16, kRegion = 16 * kPitch;
        static_assert(16 * UO % 64 == 0, "whole units a lane");
        char* region = lds + wave * kRegion;
        const long wr0 = er + wr * WF, wc0 = ec + wc * CN * 16;
#pragma unroll
        for (int j = 0; j < CN; ++j) {
#pragma unroll
          for (int i = 0; i < RM; ++i) {
            vec4<O> o;
#pragma unroll
            for (int q = 0; q < 4; ++q) o[q] = (O)acc[i][j][q];
            *reinterpret_cast<vec4<O>*>(region + lc * kPitch + (i * 16 + lr) * (int)sizeof(O)) = o;
          }
          wave_sync();
#pragma unroll 2
          for (int n = 0; n < 16 * UO / 64; ++n) {
            const int e = lane + n * 64, r = e % UO * EO;
            const long c = wc0 + j * 16 + e / UO, left = a.nr - wr0 - r;
            if (c >= a.nc || left <= 0) continue;
            Vec16<O> o;
            o.load(reinterpret_cast<const O*>(region + e / UO * kPitch + e % UO * 16));
            o.store_upto(out + c * ldo + wr0 + r, left);
          }
          wave_sync();
        }
      };
      if (a.splits == 1) finish(static_cast<T*>(which ? a.out[1] : a.out[0]), a.ldo);
      else finish(a.partial + ((long)split * problems + which) * a.nc * a.nr, a.nr);
    }
    if constexpr (!kAhead) return;
    if (!more) return;
    __syncthreads();               // the epilogue's reads of LDS are done
  }
}

// LDS of a kernel: the two buffers and the biases, or what the epilogue's regions take
template <typename T, int MODE, int BR, int BC, int WR, int WC> constexpr int lds_bytes() {
  constexpr bool kPair = MODE <= mz_gff::kGateGrad;
  constexpr int TR = kPair ? BR / 2 : BR, WF = TR / WR, units = WF * (int)sizeof(T) / 16, PR = 16 * units < 64 ? 64 / units : 16;
  constexpr int buffers = 2 * (BR + BC) * 128, region = PR * (WF * (int)sizeof(T) + 16);
  constexpr int regions = MODE == mz_gff::kForward    ? WR * WC * region
                          : MODE == mz_gff::kGateGrad ? WR * WC * (BR == 64 ? 4 : 2) * region + WC * 2 * TR * 4
                                                      : WR * WC * 16 * (WF * 4 + 16);
  static_assert(!kPair || regions <= buffers, "the biases lie behind the buffers");
  constexpr int bytes = (regions > buffers ? regions : buffers) + (kPair ? 2 * TR * 4 : 0);
  static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
  return bytes;
}
// wavefronts per SIMD that the registers have to leave room for
constexpr int min_waves(int side) { return side == 64 ? 4 : 2; }

template <typename T, int MODE, int S, int WR, int WC, int ACT>
__global__ __launch_bounds__(WR * WC * 64, min_waves(S)) void gff_gemm_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  gff_gemm<T, MODE, S, S, WR, WC, ACT>(a, blockIdx.x, gridDim.x, lds);
}
// the two products of a backward pass in one launch: the input gradient's workgroups (a multiple of 8 of each) come first,
// or the weights' where those are the longer ones (3000 x 3000 x 100 bf16 backward: 43.1 us, 45.4 with the shorter first;
// 52331 x 487 x 66: 78, 87)
template <typename T, int S, int WR, int WC>
__global__ __launch_bounds__(WR * WC * 64, min_waves(S)) void gff_both_kernel(Args x, Args w, unsigned blocks_x, unsigned blocks_w, int w_first) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const bool is_x = w_first ? blockIdx.x >= blocks_w : blockIdx.x < blocks_x;
  if (is_x) gff_gemm<T, mz_gff::kInputGrad, S, S, WR, WC, kAnyActivation>(x, w_first ? blockIdx.x - blocks_w : blockIdx.x, blocks_x, lds);
  else gff_gemm<T, mz_gff::kWeightGrad, S, S, WR, WC, kAnyActivation>(w, w_first ? blockIdx.x : blockIdx.x - blocks_x, blocks_w, lds);
}

// workgroups of a product in S x S tiles, a multiple of the 8 XCDs: one a tile, or for pair products what the chip holds (that a
// launch can have them is the choice of the tile's to see to: max_groups in gated_ff.hip)
template <int MODE, int S> long gemm_blocks(const Args& a) {
  constexpr bool kPair = MODE <= mz_gff::kGateGrad;
  constexpr int TR = kPair ? S / 2 : S;
  const long total = ((a.nr + TR - 1) / TR) * ((a.nc + S - 1) / S) * (MODE == mz_gff::kWeightGrad ? 2 : 1) * a.splits;
  const long held = (long)mz::compute_units() / 8 * 8 * (S == 256 ? 1 : S == 128 ? 2 : 4), blocks = (total + 7) / 8 * 8;
  return kPair && S != 256 && blocks > held ? held : blocks;
}

template <typename T, int MODE, int S, int WR, int WC, int ACT> int launch_kernel(const Args& a, hipStream_t s) {
  constexpr int kLds = lds_bytes<T, MODE, S, S, WR, WC>();
  static bool done[mz::kMaxDevices] = {false};
  const auto kernel = gff_gemm_kernel<T, MODE, S, WR, WC, ACT>;
  if (int rc = mz::ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), kLds, done, "mz_gated_ff")) return rc;
  const long blocks = gemm_blocks<MODE, S>(a);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(WR * WC * 64), kLds, s, a);
  return MZ_OK;
}
template <typename T, int MODE, int S, int WR, int WC> int launch_one(const Args& a, hipStream_t s) {
  if constexpr (MODE == mz_gff::kGateGrad) {
    switch (a.activation) {
      case mz_gff::kSilu: return launch_kernel<T, MODE, S, WR, WC, mz_gff::kSilu>(a, s);
      case mz_gff::kGelu: return launch_kernel<T, MODE, S, WR, WC, mz_gff::kGelu>(a, s);
      case mz_gff::kRelu: return launch_kernel<T, MODE, S, WR, WC, mz_gff::kRelu>(a, s);
      default: return launch_kernel<T, MODE, S, WR, WC, mz_gff::kSigmoid>(a, s);
    }
  } else {
    return launch_kernel<T, MODE, S, WR, WC, kAnyActivation>(a, s);
  }
}
template <typename T, int MODE> int launch_mode(const Args& a, int tile, hipStream_t s) {
  // float32's matrix instructions are slow enough for the smaller tiles to keep up with (18432 x 256 x 1024 forward: 128 x
  // 128 tiles 160 us, 64 x 64 172)
  if constexpr (sizeof(T) == 2)
    if (tile == 0) return launch_one<T, MODE, 256, 2, 4>(a, s);
  if (tile <= 1) return launch_one<T, MODE, 128, 2, 2>(a, s);
  return launch_one<T, MODE, 64, 2, 2>(a, s);
}
template <typename T> int launch_any(const Args& a, int mode, int tile, hipStream_t s) {
  switch (mode) {
    case mz_gff::kForward: return launch_mode<T, mz_gff::kForward>(a, tile, s);
    case mz_gff::kGateGrad: return launch_mode<T, mz_gff::kGateGrad>(a, tile, s);
    case mz_gff::kInputGrad: return launch_mode<T, mz_gff::kInputGrad>(a, tile, s);
    default: return launch_mode<T, mz_gff::kWeightGrad>(a, tile, s);
  }
}
template <typename T, int S> int launch_both_in(const Args& x, const Args& w, hipStream_t s) {
  constexpr int kLds = lds_bytes<T, mz_gff::kInputGrad, S, S, 2, 2>();
  static bool done[mz::kMaxDevices] = {false};
  const auto kernel = gff_both_kernel<T, S, 2, 2>;
  if (int rc = mz::ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), kLds, done, "mz_gated_ff")) return rc;
  const long bx = gemm_blocks<mz_gff::kInputGrad, S>(x), bw = gemm_blocks<mz_gff::kWeightGrad, S>(w);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(bx + bw)), dim3(256), kLds, s, x, w, (unsigned)bx, (unsigned)bw,
                     w.steps_per_split > x.steps_per_split ? 1 : 0);
  return MZ_OK;
}
template <typename T> int launch_both(const Args& x, const Args& w, int tile, hipStream_t s) {
  return tile == 1 ? launch_both_in<T, 128>(x, w, s) : launch_both_in<T, 64>(x, w, s);
}

// ---- a few tokens (at most 16): the weights are read once, straight into the matrix instructions' registers; 16
// features (their gate and up rows) a workgroup, its four wavefronts split k and add up through LDS.
template <typename T> __global__ __launch_bounds__(256) void gff_few_kernel(Args a) {
  constexpr int EC = 16 / (int)sizeof(T), KB = 4 * EC;     // k of one round of a wavefront's lanes
  constexpr int kUnroll = 4;
  __shared__ f32x4 red[3][2][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l = lane & 15;
  const long f0 = (long)blockIdx.x * 16;
  // rows and tokens past the end read the last one's: their results are not stored
  const long f_row = f0 + l < a.nr ? f0 + l : a.nr - 1, c_row = l < a.nc ? l : a.nc - 1;
  const T* wg = static_cast<const T*>(a.r[0]) + f_row * a.ldr;
  const T* wu = static_cast<const T*>(a.r[1]) + f_row * a.ldr;
  const T* x = static_cast<const T*>(a.c[0]) + c_row * a.ldc;
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  const int rounds = (int)((a.nk + KB - 1) / KB);
  for (int q0 = wave * kUnroll; q0 < rounds; q0 += 4 * kUnroll) {
    Vec16<T> rg[kUnroll], ru[kUnroll], cf[kUnroll];
    if ((long)(q0 + kUnroll) * KB <= a.nk) {        // all of it inside: loads without conditions, all in flight
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const long k = (long)(q0 + q) * KB + g * EC;
        rg[q].load(wg + k);
        ru[q].load(wu + k);
        cf[q].load(x + k);
      }
    } else {
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const long k = (long)(q0 + q) * KB + g * EC;
        rg[q].load_upto(wg + k, a.nk - k);
        ru[q].load_upto(wu + k, a.nk - k);
        cf[q].load_upto(x + k, a.nk - k);
      }
    }
#pragma unroll
    for (int q = 0; q < kUnroll; ++q) {
      const u32x4 c = __builtin_bit_cast(u32x4, cf[q].v);
      acc[0] = mma(__builtin_bit_cast(u32x4, rg[q].v), c, acc[0], T{});
      acc[1] = mma(__builtin_bit_cast(u32x4, ru[q].v), c, acc[1], T{});
    }
  }
  if (wave > 0) {
    red[wave - 1][0][lane] = acc[0];
    red[wave - 1][1][lane] = acc[1];
  }
  __syncthreads();
  if (wave > 0 || l >= a.nc) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    acc[0] += red[w][0][lane];
    acc[1] += red[w][1][lane];
  }
  const T* bg = static_cast<const T*>(a.bias[0]);
  const T* bu = static_cast<const T*>(a.bias[1]);
  T* out = static_cast<T*>(a.out[0]) + l * a.ldo;
  with_activation<kAnyActivation>(a.activation, [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long f = f0 + g * 4 + q;
      if (f >= a.nr) continue;
      const float gate = acc[0][q] + (bg ? (float)bg[f] : 0.f), up = acc[1][q] + (bu ? (float)bu[f] : 0.f);
      out[f] = (T)(activate<T, decltype(kind)::value>(gate) * up);
    }
  });
}

template <typename T> int launch_few(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((gff_few_kernel<T>), dim3((unsigned)((a.nr + 15) / 16)), dim3(256), 0, s, a);
  return MZ_OK;
}

}  // namespace
#endif  // MZ_GFF_KERNELS
