// Gated feed-forward projection, forward and backward:
//     g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u                    x [M][K], Wg, Wu [F][K], h [M][F]
//     dg = dh u act'(g),  du = dh act(g)
//     dx = dg Wg + du Wu,   dWg = dg^T x,  dWu = du^T x,   dbg = sum_rows dg,  dbu = sum_rows du
// Forward is one kernel: a wavefront owns the gate and the up product of the same features, so activation and product
// happen in its registers and only h is written.  Nothing else is kept for the backward pass: it computes g and u again, writes
// dg and du in the operands' type - they are matrix operands next - and runs the two products that need them.  Computing them
// again takes no memory and rounds neither; in time, 4 M K F operations against 8 M F bytes of 16 bits (16 of float32) written
// and read, it is the cheaper way up to a K of about 500 in 16 bits (1000 against values kept in float32) and 120 in float32
// and the dearer one above: about 430 of the gate gradient's 484 us at 8192 x 2048 x 8192 bf16, 160 of 178 at 18432 x 256 x
// 1024 float32.
// What rounding dg and du to 16 bits costs: every term of dx and dW is off by its own relative error, independent of the others', so
// the sums are off by that error relative to their own size however long they are; with the result's rounding, as large, that
// is sqrt(2) of it (relative RMS 2.35e-3 in bf16 and 2.9e-4 in f16 against 1.66e-3 and 2.1e-4, measured from 32 x 256 x 256
// to 18432 x 256 x 1024 alike).  A second operand that holds what the rounding left takes that away and doubles the products'
// steps.  It is carried where a pass is bound by its launches and that is all but free, see make_plan().  Sums
// over few tiles are split along k into float32 partial results that a second launch adds up in a fixed order: no atomics,
// the same bits on every run.
#include "gated_ff.h"

#include <algorithm>

namespace {

using mz_gff::Args;

int elem_bytes(int dtype) { return dtype == MZ_F32 ? 4 : 2; }
int unit_elems(int dtype) { return 16 / elem_bytes(dtype); }
int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int launch(const Args& a, int dtype, int mode, int tile, hipStream_t s) {
  return dtype == MZ_F32 ? mz_gff::launch_f32(a, mode, tile, s)
         : dtype == MZ_BF16 ? mz_gff::launch_bf16(a, mode, tile, s)
                            : mz_gff::launch_f16(a, mode, tile, s);
}

int launch_both(const Args& x, const Args& w, int dtype, int tile, hipStream_t s) {
  return dtype == MZ_F32 ? mz_gff::launch_both_f32(x, w, tile, s)
         : dtype == MZ_BF16 ? mz_gff::launch_both_bf16(x, w, tile, s)
                            : mz_gff::launch_both_f16(x, w, tile, s);
}

// What is left of a backward pass, in one launch: cut sums joined - out[p][c][r] = sum over the splits of
// partial[split][p][c][r] - and the bias gradients, dbias[side][f] = sum over the token tiles of col[tile][side][f].
struct Join {
  const float* partial;
  long n, per_problem;       // elements of all problems, of one
  int splits;
  void* out[2];
  unsigned blocks;
};
struct Finish {
  Join join[2];
  const float* col;
  long tiles, F;
  void* dbias[2];
  unsigned bias_blocks;
};

template <typename T> __device__ __forceinline__ void join_part(const Join& j, unsigned block) {
  T* out0 = static_cast<T*>(j.out[0]);
  T* out1 = static_cast<T*>(j.out[1]);
  for (long i = ((long)block * 256 + threadIdx.x) * 4; i < j.n; i += (long)j.blocks * 1024) {
    const int m = (int)(j.n - i < 4 ? j.n - i : 4);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < j.splits; ++s) {           // rows of odd lengths start anywhere: a vector of float's alignment
      Vec16<float> t;
      t.load_upto(j.partial + s * j.n + i, m);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += t.v[q];
    }
    for (int q = 0; q < m; ++q) {
      const long e = i + q;
      if (e < j.per_problem) out0[e] = (T)v[q];
      else out1[e - j.per_problem] = (T)v[q];
    }
  }
}

template <typename T> __global__ __launch_bounds__(256) void finish_kernel(Finish f) {
  __shared__ float red[2][32][9];
  unsigned b = blockIdx.x;
  if (b < f.join[0].blocks) return join_part<T>(f.join[0], b);
  b -= f.join[0].blocks;
  if (b < f.join[1].blocks) return join_part<T>(f.join[1], b);
  b -= f.join[1].blocks;
  const int col = threadIdx.x & 7, lane = threadIdx.x >> 3;             // 8 features, 32 tile lanes
  const long c = (long)b * 8 + col;
  float g = 0.f, u = 0.f;
  if (c < f.F) {
    for (long t0 = lane; t0 < f.tiles; t0 += 32 * 4) {                  // eight loads in flight
      float v[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long t = t0 + 32 * i;
        v[0][i] = t < f.tiles ? f.col[(t * 2 + 0) * f.F + c] : 0.f;
        v[1][i] = t < f.tiles ? f.col[(t * 2 + 1) * f.F + c] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g += v[0][i];
        u += v[1][i];
      }
    }
  }
  red[0][lane][col] = g;
  red[1][lane][col] = u;
  __syncthreads();
  if (lane >= 2 || c >= f.F) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) v += red[lane][k][col];
  T* out = static_cast<T*>(f.dbias[lane]);
  if (out) out[c] = (T)v;
}

Join make_join(const Args& a, int problems) {
  const long n = a.nr * a.nc * problems, want = (n + 1023) / 1024, cap = 8L * mz::compute_units();
  return {a.partial, n, a.nr * a.nc, a.splits, {a.out[0], a.out[1]}, (unsigned)(want < cap ? want : cap)};
}
void finish(const Finish& f, int dtype, hipStream_t s) {
  const dim3 grid(f.join[0].blocks + f.join[1].blocks + f.bias_blocks);
  if (grid.x == 0) return;
  if (dtype == MZ_F32) hipLaunchKernelGGL((finish_kernel<float>), grid, dim3(256), 0, s, f);
  else if (dtype == MZ_BF16) hipLaunchKernelGGL((finish_kernel<__bf16>), grid, dim3(256), 0, s, f);
  else hipLaunchKernelGGL((finish_kernel<_Float16>), grid, dim3(256), 0, s, f);
}

int64_t tiles(int64_t nr, int64_t nc, int tr, int bc) { return ((nr + tr - 1) / tr) * ((nc + bc - 1) / bc); }

// Tile and split of a product launched by itself, by its estimated time (microseconds).  A tile's workgroups share a compute unit `at_once`
// at a time; a step of one takes `alone`, and no less than `shared` times the workgroups there; `ends` is what a round
// costs besides its steps (first loads, epilogue), by mode.  A sum cut into parts costs another launch and its partial
// results' way through memory.  Measured per step (64 16-bit or 32 float32 values of k), one workgroup alone / the
// compute unit full, on products of one to 4096 tiles; the estimate is within a fifth of what it was fitted to, and
// choosing by it within a tenth of the best of all choices (18432 x 256 x 1024, dx: 128 x 128 tiles 29 us, 64 x 64 39,
// 256 x 256 40; 1000 x 256 x 1000 float32, dx: 64 x 64 in 8 parts 17 us, whole 46, 128 x 128 in 16 parts 19, whole 138).
struct TileCost {
  int at_once;
  float alone, shared, ends[3];                    // ends: kForward, kGateGrad, the plain products
};
constexpr TileCost kCost16[3] = {{1, 1.4f, 1.45f, {7.f, 14.f, 8.f}}, {2, .58f, .5f, {3.5f, 6.f, 4.5f}}, {5, .34f, .23f, {2.2f, 4.5f, 2.5f}}};
constexpr TileCost kCost32[3] = {{}, {2, 2.1f, 1.95f, {4.f, 8.f, 5.f}}, {5, .72f, .53f, {2.5f, 4.f, 3.f}}};

struct Split {
  int tile, splits, steps;
  float time;
  int64_t groups;                                  // workgroups
};
constexpr int kMaxSplits = 32, kCus = 256;         // of an MI355X: the choice, and with it a sum's order, is the same everywhere

const TileCost& cost_of(int dtype, int tile) { return (dtype == MZ_F32 ? kCost32 : kCost16)[tile]; }
float join_time(int64_t elements, int splits) { return splits > 1 ? (float)elements * splits * 8.f / 8e6f : 0.f; }

// Workgroups that a launch can have: HIP counts its threads in 32 bits (16 less, for rounding up to all XCDs).  The pair products'
// workgroups in the smaller tiles are as many as the chip holds; their tiles are numbered in 32 bits.
int64_t max_groups(int tile, bool pair) { return pair && tile != 0 ? 0x3ffffff0ll : (1ll << 32) / (tile == 0 ? 512 : 256) - 16; }

// f(the product of nr x nc results, `problems` of them, in `tile` with its sum cut into 1, 2, 3 .. parts)
template <typename Fn> void for_cuts(int64_t nr, int64_t nc, int64_t steps, int tile, int problems, bool pair, Fn&& f) {
  const int side = mz_gff::tile_side(tile);
  const int64_t whole = tiles(nr, nc, pair ? side / 2 : side, side) * problems;
  for (int want = 1; want <= (pair ? 1 : kMaxSplits); want += want < 4 ? 1 : want < 8 ? 2 : want < 16 ? 4 : 8) {
    if (want > 1 && want > steps / 2) break;
    const int64_t per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
    if (whole * splits > max_groups(tile, pair)) break;
    f(Split{tile, (int)splits, (int)per, 0.f, whole * splits});
  }
}

// the estimated time of `elements` results in the tiles and the cut of s, in a launch of their own
float time_alone(const Split& s, int64_t elements, int dtype, int mode) {
  const TileCost& c = cost_of(dtype, s.tile);
  const int64_t share = (s.groups + kCus - 1) / kCus, rounds = share / c.at_once, rest = share % c.at_once;
  auto round = [&](int64_t n) {
    const float step = c.shared * n > c.alone ? c.shared * n : c.alone;
    return s.steps * step + c.ends[mode < 2 ? mode : 2];
  };
  return rounds * round(c.at_once) + (rest ? round(rest) : 0.f) + (s.splits > 1 ? 3.f + join_time(elements, s.splits) : 0.f);
}

Split pick(int64_t nr, int64_t nc, int64_t steps, int dtype, int mode, int only = -1) {
  const bool pair = mode <= mz_gff::kGateGrad;
  const int problems = mode == mz_gff::kWeightGrad ? 2 : 1;
  Split best = {2, 1, (int)steps, -1.f, 0};        // stays where no tile is large enough: refused before anything is launched
  for (int t = dtype == MZ_F32 ? 1 : 0; t < 3; ++t) {
    if (only >= 0 && t != only) continue;
    for_cuts(nr, nc, steps, t, problems, pair, [&](Split s) {
      s.time = time_alone(s, nr * nc * problems, dtype, mode);
      if (best.time < 0.f || s.time < best.time) best = s;
    });
  }
  if (best.time < 0.f) best.time = 1e30f;
  return best;
}

// Two products in one launch, the longer workgroups first and the others where those leave room: the larger of two
// estimates.  One is all steps at the compute units' full rate - less of it while fewer than `at_once` share one - with part of
// the ends and of the last workgroups; the other the compute unit with most steps, if all workgroups are there at once.
// Fitted to 62 backward passes of all sizes with 40 to 126 pairs of cuts each: what this and pick() choose - separate
// launches, which alone have the largest tiles, where that is estimated faster - is within 3 % of the best on average, one
// launch only where a single round holds both within 6 % (18432 x 256 x 1024 bf16: 71 us then, 48 now; 3000 x 3000 x 100:
// 32, 19).  The worst that the choice was seen to lose: 4553 x 1505 x 218 float32, backward 193 us, with dw cut in 12 parts and
// not in 6 179.
float time_together(const TileCost& c, const Split& x, const Split& w) {
  const int64_t n = x.groups + w.groups, most = (n + kCus - 1) / kCus, x_most = (x.groups + kCus - 1) / kCus;
  const float at_once = (float)c.at_once, held = n <= kCus ? 1.f : n >= kCus * c.at_once ? at_once : (float)n / kCus;
  auto rate = [&](float h) { return c.shared * (1.f + .4f * (1.f - h / at_once)); };     // a step's time, of h together
  const int longer = x.steps > w.steps ? x.steps : w.steps, shorter = x.steps + w.steps - longer;
  const float last = shorter * (c.shared * held > c.alone ? c.shared * held : c.alone) + c.ends[2];
  const float all = ((x.groups * x.steps + w.groups * w.steps) * rate(held) + n * c.ends[2] * .35f) / kCus + .25f * last;
  float one = longer * rate(at_once) * at_once;
  if (most <= c.at_once) {
    const int64_t l0 = x_most * x.steps + (most - x_most) * w.steps, l1 = l0 - x.steps + w.steps;
    one = (l0 > l1 ? l0 : l1) * rate((float)most);
  }
  if (one < longer * c.alone) one = longer * c.alone;
  one += c.ends[2];
  return all > one ? all : one;
}

struct Shape {
  int64_t M, K, F, Fp;       // Fp: F in whole 16-byte units, the row length of dg and du
  int dtype;
  bool ragged;               // K is no whole number of units: a row's last unit reaches into the next row, the last row's
                             // past the end (gated_ff.h: nk_all)
  int step() const { return 128 / elem_bytes(dtype); }
  int64_t steps(int64_t nk) const { return nk > 0 ? (nk + step() - 1) / step() : 1; }
  // the rows at a matrix's end from which a unit that starts inside a row of K would reach past the last one
  int64_t end_rows() const { return ragged ? (round_up(K, unit_elems(dtype)) - K + K - 1) / K : 0; }
  // the k that the steps take: of K (forward), of F (input gradient) and of M (weight gradient); what is left is less
  // than a unit of K, less than two of F (end_rows() and what makes whole units before it) and less than one of M
  int64_t nk_K() const { return K / unit_elems(dtype) * unit_elems(dtype); }
  int64_t nk_F() const { return !ragged ? F : F > end_rows() ? (F - end_rows()) / unit_elems(dtype) * unit_elems(dtype) : 0; }
  int64_t nk_M() const { return M > end_rows() ? M - end_rows() : 0; }
};
Shape make_shape(int64_t M, int64_t K, int64_t F, int dtype) {
  const int e = unit_elems(dtype);
  return {M, K, F, round_up(F, e), dtype, K % e != 0};
}
// Tokens the streaming kernel takes: at 16, 2048 x 2048 bf16 8.3 us (64 x 64 tiles 12.3), 1000 x 5000 float32 13.6
// (23.2), 4096 x 16384 bf16 out of the caches 47 (42); at 32, with two blocks of tokens, 9.8 (12.0), 19.9 (23.6), 59 (43).
constexpr int64_t kFew = 16;

struct Backward {
  Split dx, dw;              // asked for together
  Split dx_only, dw_only;    // one without the other
  int parts;                 // of dg and du (Args::parts)
  bool both;                 // the two products in one launch, in the same tiles
  int gate_tile;
  int64_t dgu_bytes, col_bytes, partial_bytes;     // partial results of cut sums: dx's and then dw's
  int64_t bytes() const { return 2 * parts * dgu_bytes + col_bytes + partial_bytes; }
};
int64_t partial_bytes(const Split& s, int64_t elements) { return s.splits > 1 ? round_up(s.splits * elements * 4, 256) : 0; }

Backward make_plan(const Shape& h) {
  Backward b;
  // Second parts of dg and du in the 16-bit types (above) where they cost 0 to 4 us: kernels of the backward pass without / with them
  // 32 x 256 x 256 12.3 / 12.0 us, 90 x 64 x 72 10.9 / 11.8, 8000 x 256 x 1 15.2 / 17.5, 4 x 1024 x 2048 19.4 / 23.4.  Past these
  // limits they cost the products' time again: 128 x 256 x 1024 13.1 / 15.0, 1000 x 250 x 700 22.7 / 30.1, 1024 x 256 x 1024
  // 22.7 / 34.2, and the weights' second reading 1 x 4096 x 8192 77.8 / 127.4.
  b.parts = h.dtype != MZ_F32 && h.M * h.F <= 8192 && h.K * h.F <= 1 << 21 ? 2 : 1;
  const int only = b.parts == 2 ? 2 : -1;          // in the smallest tiles
  const Split gate = pick(h.F, h.M, h.steps(h.nk_K()), h.dtype, mz_gff::kGateGrad, only);
  b.gate_tile = gate.groups ? gate.tile : -1;
  const int64_t fs = 2 * b.parts * h.steps(h.nk_F()), ms = b.parts * h.steps(h.nk_M());
  b.dx = b.dx_only = pick(h.K, h.M, fs, h.dtype, mz_gff::kInputGrad, only);
  b.dw = b.dw_only = pick(h.K, h.F, ms, h.dtype, mz_gff::kWeightGrad, only);
  b.both = false;
  float least = b.dx.time + b.dw.time + 9.f;       // and a launch more
  // Against launches in the largest tiles, which a shared one does not have, it has to win by more than the estimate is off by
  // (46984 x 2394 x 166 bf16: estimated 0.96 of the separate launches' time, measured 1.08).
  if (b.dx.tile == 0 || b.dw.tile == 0) least *= .94f;
  for (int t = b.parts; t < 3; ++t)                // parts: the smallest tiles only; the largest has no kernel of both
    for_cuts(h.K, h.M, fs, t, 1, false, [&](const Split& x) {
      for_cuts(h.K, h.F, ms, t, 2, false, [&](const Split& w) {
        if (x.groups + w.groups > max_groups(t, false)) return;
        const float time = time_together(cost_of(h.dtype, t), x, w) + join_time(h.M * h.K, x.splits) + join_time(2 * h.F * h.K, w.splits);
        if (time >= least) return;
        b.both = true;
        least = time;
        b.dx = x;
        b.dw = w;
      });
    });
  // A gradient that is asked for without the other (frozen weights, an input without a gradient) has the cut that it has with
  // it, and so the same bits, unless its own is estimated clearly faster (46984 x 2394 x 166 bf16, dw: 110 us, cut for the shared
  // launch 180; 7517 x 3248 x 209 float32, dw: 218, 317; 18432 x 256 x 1024 float32, dx: 171, 254).
  const auto clearly = [&](const Split& own, const Split& joint, int64_t elements, int mode) {
    const float t = time_alone(joint, elements, h.dtype, mode);
    return own.time < .9f * t && own.time < t - 4.f;           // by more than a launch
  };
  if (!clearly(b.dx_only, b.dx, h.M * h.K, mz_gff::kInputGrad)) b.dx_only = b.dx;
  if (!clearly(b.dw_only, b.dw, 2 * h.F * h.K, mz_gff::kWeightGrad)) b.dw_only = b.dw;
  b.dgu_bytes = round_up(h.M * h.Fp * elem_bytes(h.dtype), 256);
  const int side = mz_gff::tile_side(b.gate_tile < 0 ? 2 : b.gate_tile);
  b.col_bytes = round_up((h.M + side - 1) / side * 2 * h.F * 4, 256);
  const int64_t only_bytes = std::max(partial_bytes(b.dx_only, h.M * h.K), partial_bytes(b.dw_only, 2 * h.F * h.K));
  b.partial_bytes = std::max(partial_bytes(b.dx, h.M * h.K) + partial_bytes(b.dw, 2 * h.F * h.K), only_bytes);
  return b;
}

// Weighing all pairs of cuts takes 4 us of the host, several times a training step of the same few sizes: each thread keeps
// the plans of sizes it has met.
Backward plan_backward(const Shape& h) {
  struct Kept {
    int64_t M = 0, K = 0, F = 0;                   // no plan has M = 0
    int dtype = 0;
    Backward plan;
  };
  thread_local Kept kept[16];
  Kept& k = kept[(uint64_t)(h.M * 31 + h.K * 17 + h.F * 7 + h.dtype) % 16];
  if (k.M != h.M || k.K != h.K || k.F != h.F || k.dtype != h.dtype) {
    k.plan = make_plan(h);
    k.M = h.M; k.K = h.K; k.F = h.F; k.dtype = h.dtype;
  }
  return k.plan;
}

int check_shape(const char* who, int64_t M, int64_t K, int64_t F, int32_t dtype, int32_t activation) {
  MZ_REQUIRE(dtype == MZ_F32 || dtype == MZ_BF16 || dtype == MZ_F16, "%s: unknown element type %d", who, dtype);
  MZ_REQUIRE(M > 0 && K > 0 && F > 0 && K <= (1 << 20) && F <= (1 << 20) && M <= (1ll << 36),
             "%s: sizes out of range (M = %lld, K = %lld, F = %lld; M up to 2^36, K and F up to 2^20)", who, (long long)M, (long long)K,
             (long long)F);
  MZ_REQUIRE(activation >= 0 && activation <= mz_gff::kSigmoid, "%s: unknown activation %d", who, activation);
  return MZ_OK;
}
int check_tiles(const char* who, bool fits) {
  MZ_REQUIRE(fits, "%s: too many output tiles for a launch", who);
  return MZ_OK;
}
int check_stride(const char* who, const Shape& h, int64_t ldx) {
  MZ_REQUIRE(ldx >= h.K && ldx <= (1 << 22) / elem_bytes(h.dtype),
             "%s: stride of x out of range (%lld, K = %lld; rows up to 4 MiB apart)", who, (long long)ldx, (long long)h.K);
  return MZ_OK;
}

}  // namespace

extern "C" {

int64_t mz_gated_ff_workspace_bytes(int64_t M, int64_t K, int64_t F, int32_t dtype, int32_t backward) {
  if (check_shape("mz_gated_ff_workspace_bytes", M, K, F, dtype, 0)) return -1;
  if (!backward) return 0;
  return plan_backward(make_shape(M, K, F, dtype)).bytes();
}

int mz_gated_ff_plan(int64_t M, int64_t K, int64_t F, int32_t dtype, int32_t want_dx, int32_t want_dw, int32_t* plan) {
  MZ_REQUIRE(plan, "mz_gated_ff_plan: null plan");
  if (int rc = check_shape("mz_gated_ff_plan", M, K, F, dtype, 0)) return rc;
  const Shape sh = make_shape(M, K, F, dtype);
  const Backward b = plan_backward(sh);
  const Split fwd = pick(F, M, sh.steps(sh.nk_K()), dtype, mz_gff::kForward);
  const Split &dx = want_dw ? b.dx : b.dx_only, &dw = want_dx ? b.dw : b.dw_only;
  if (int rc = check_tiles("mz_gated_ff_plan", fwd.groups && b.gate_tile >= 0 && (!want_dx || dx.groups) && (!want_dw || dw.groups))) return rc;
  plan[0] = M <= kFew ? 0 : mz_gff::tile_side(fwd.tile);
  plan[1] = mz_gff::tile_side(b.gate_tile);
  plan[2] = want_dx ? mz_gff::tile_side(dx.tile) : 0;
  plan[3] = want_dx ? dx.splits : 0;
  plan[4] = want_dw ? mz_gff::tile_side(dw.tile) : 0;
  plan[5] = want_dw ? dw.splits : 0;
  plan[6] = b.both && want_dx && want_dw;
  plan[7] = b.parts;
  return MZ_OK;
}

int mz_gated_ff_fwd(const void* x, int64_t ldx, const void* w_gate, const void* w_up, const void* b_gate, const void* b_up,
                    int64_t M, int64_t K, int64_t F, int32_t dtype, int32_t activation, void* h, void* workspace,
                    int64_t workspace_bytes, mz_stream_t stream) {
  MZ_REQUIRE(x && w_gate && w_up && h, "mz_gated_ff_fwd: null tensor");
  if (int rc = check_shape("mz_gated_ff_fwd", M, K, F, dtype, activation)) return rc;
  const Shape sh = make_shape(M, K, F, dtype);
  if (int rc = check_stride("mz_gated_ff_fwd", sh, ldx)) return rc;
  hipStream_t s = mz::as_stream(stream);
  Args a = {};
  a.r[0] = w_gate; a.r[1] = w_up;
  a.c[0] = a.c[1] = x;
  a.ldr = K; a.ldc = ldx;
  a.nr = F; a.nc = M; a.nk = M <= kFew ? K : sh.nk_K(); a.nk_all = K;
  a.out[0] = h; a.ldo = F;
  a.bias[0] = b_gate; a.bias[1] = b_up;
  a.activation = activation;
  a.splits = 1;
  if (M <= kFew) {
    if (int rc = dtype == MZ_F32 ? mz_gff::launch_few_f32(a, s) : dtype == MZ_BF16 ? mz_gff::launch_few_bf16(a, s) : mz_gff::launch_few_f16(a, s))
      return rc;
    return mz::check_launch("mz_gated_ff_fwd");
  }
  a.steps_per_split = (int)sh.steps(a.nk);
  const Split cut = pick(F, M, sh.steps(a.nk), dtype, mz_gff::kForward);
  if (int rc = check_tiles("mz_gated_ff_fwd", cut.groups > 0)) return rc;
  if (int rc = launch(a, dtype, mz_gff::kForward, cut.tile, s)) return rc;
  return mz::check_launch("mz_gated_ff_fwd");
}

int mz_gated_ff_bwd(const void* x, int64_t ldx, const void* w_gate, const void* w_up, const void* b_gate, const void* b_up,
                    const void* dh, int64_t M, int64_t K, int64_t F, int32_t dtype, int32_t activation, void* dx,
                    void* dw_gate, void* dw_up, void* db_gate, void* db_up, void* workspace, int64_t workspace_bytes,
                    mz_stream_t stream) {
  MZ_REQUIRE(x && w_gate && w_up && dh, "mz_gated_ff_bwd: null tensor");
  MZ_REQUIRE((dw_gate == nullptr) == (dw_up == nullptr), "mz_gated_ff_bwd: dw_gate and dw_up go together");
  MZ_REQUIRE(dx || dw_gate || db_gate || db_up, "mz_gated_ff_bwd: no gradient asked for");
  if (int rc = check_shape("mz_gated_ff_bwd", M, K, F, dtype, activation)) return rc;
  const Shape sh = make_shape(M, K, F, dtype);
  if (int rc = check_stride("mz_gated_ff_bwd", sh, ldx)) return rc;
  const Backward plan = plan_backward(sh);
  const int64_t need = plan.bytes();
  MZ_REQUIRE(workspace && workspace_bytes >= need && (size_t)workspace % 16 == 0,
             "mz_gated_ff_bwd: workspace too small (%lld of %lld bytes) or not 16-byte aligned", (long long)workspace_bytes,
             (long long)need);
  const Split &cut_x = dw_gate ? plan.dx : plan.dx_only, &cut_w = dx ? plan.dw : plan.dw_only;
  if (int rc = check_tiles("mz_gated_ff_bwd", plan.gate_tile >= 0 && (!dx || cut_x.groups) && (!dw_gate || cut_w.groups))) return rc;
  hipStream_t s = mz::as_stream(stream);
  char* dg = static_cast<char*>(workspace);
  char* du = dg + plan.dgu_bytes;
  char* behind = dg + 2 * plan.parts * plan.dgu_bytes;   // dg, du [, dg_lo, du_lo]
  float* cols = reinterpret_cast<float*>(behind);
  char* partial = behind + plan.col_bytes;
  const bool biases = db_gate || db_up;

  Args a = {};                                     // dg, du
  a.r[0] = w_gate; a.r[1] = w_up;
  a.c[0] = a.c[1] = x;
  a.ldr = K; a.ldc = ldx;
  a.nr = F; a.nc = M; a.nk = sh.nk_K(); a.nk_all = K;
  a.out[0] = dg; a.out[1] = du; a.ldo = sh.Fp;
  a.parts = plan.parts;
  if (plan.parts == 2) { a.out[2] = du + plan.dgu_bytes; a.out[3] = du + 2 * plan.dgu_bytes; }
  a.bias[0] = b_gate; a.bias[1] = b_up;
  a.dh = dh; a.lddh = F;
  a.col_partial = biases ? cols : nullptr;
  a.nr_pad = sh.Fp;
  a.activation = activation;
  a.splits = 1;
  a.steps_per_split = (int)sh.steps(a.nk);
  if (int rc = launch(a, dtype, mz_gff::kGateGrad, plan.gate_tile, s)) return rc;
  Args p = {}, q = {};                             // dx; dw
  p.r[0] = w_gate; p.r[1] = w_up;
  p.c[0] = dg; p.c[1] = du; p.c[2] = a.out[2]; p.c[3] = a.out[3];
  p.parts = plan.parts;
  p.ldr = K; p.ldc = sh.Fp;
  p.nr = K; p.nc = M; p.nk = sh.nk_F(); p.nk_all = F;
  p.out[0] = p.out[1] = dx; p.ldo = K;
  p.partial = reinterpret_cast<float*>(partial);
  p.splits = cut_x.splits; p.steps_per_split = cut_x.steps;
  q.r[0] = q.r[1] = x;
  q.c[0] = dg; q.c[1] = du; q.c[2] = a.out[2]; q.c[3] = a.out[3];
  q.parts = plan.parts;
  q.ldr = ldx; q.ldc = sh.Fp;
  q.nr = K; q.nc = F; q.nk = sh.nk_M(); q.nk_all = M;
  q.out[0] = dw_gate; q.out[1] = dw_up; q.ldo = K;
  q.partial = reinterpret_cast<float*>(partial + (dx ? partial_bytes(cut_x, M * K) : 0));
  q.splits = cut_w.splits; q.steps_per_split = cut_w.steps;
  if (plan.both && dx && dw_gate) {
    if (int rc = launch_both(p, q, dtype, plan.dx.tile, s)) return rc;
  } else {
    if (dx)
      if (int rc = launch(p, dtype, mz_gff::kInputGrad, cut_x.tile, s)) return rc;
    if (dw_gate)
      if (int rc = launch(q, dtype, mz_gff::kWeightGrad, cut_w.tile, s)) return rc;
  }
  Finish f = {};
  if (dx && p.splits > 1) f.join[0] = make_join(p, 1);
  if (dw_gate && q.splits > 1) f.join[1] = make_join(q, 2);
  if (biases) {
    const int side = mz_gff::tile_side(plan.gate_tile);
    f.col = cols;
    f.tiles = (M + side - 1) / side;
    f.F = F;
    f.dbias[0] = db_gate; f.dbias[1] = db_up;
    f.bias_blocks = (unsigned)((F + 7) / 8);
  }
  finish(f, dtype, s);
  return mz::check_launch("mz_gated_ff_bwd");
}

}  // extern "C"
