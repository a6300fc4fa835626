// Gated feed-forward projection, forward and backward:
//     g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u                    x [M][K], Wg, Wu [F][K], h [M][F]
//     dg = dh u act'(g),  du = dh act(g)
//     dx = dg Wg + du Wu,   dWg = dg^T x,  dWu = du^T x,   dbg = sum_rows dg,  dbu = sum_rows du
// Forward is one kernel: a wavefront owns the gate and the up product of the same features, so activation and product
// happen in its registers and only h is written.  Nothing else is kept for the backward pass: it computes g and u again
// (4 M K F operations against 8 M F bytes written and read back in 16 bits - and without rounding g and u), writes
// dg and du in the operands' type - they are matrix operands next, and their rounding adds one half step to a sum's
// terms - and runs the two products that need them.  Sums over few tiles are split along k into float32 partial
// results that a second launch adds up in a fixed order: no atomics, the same bits on every run.
#include "gated_ff.h"

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

// out[p][c][r] = sum over the splits of partial[split][p][c][r]
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ partial, int splits, long per_problem,
                                                   int problems, T* out0, T* out1) {
  const long n = per_problem * problems;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long)gridDim.x * 1024) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const int m = (int)(n - i < 4 ? n - i : 4);
    for (int s = 0; s < splits; ++s) {
      const float* p = partial + s * n + i;
      if (m == 4 && (n & 3) == 0) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
      } else {
        for (int j = 0; j < m; ++j) v[j] += p[j];
      }
    }
    for (int j = 0; j < m; ++j) {
      const long e = i + j;
      if (e < per_problem) out0[e] = (T)v[j];
      else out1[e - per_problem] = (T)v[j];
    }
  }
}
template <typename T> void join_t(const Args& a, int problems, hipStream_t s) {
  const long n = a.nr * a.nc * problems, want = (n + 1023) / 1024, cap = 8L * mz::compute_units();
  hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, s, a.partial, a.splits,
                     a.nr * a.nc, problems, static_cast<T*>(a.out[0]), static_cast<T*>(a.out[1]));
}
void join(const Args& a, int problems, int dtype, hipStream_t s) {
  if (dtype == MZ_F32) join_t<float>(a, problems, s);
  else if (dtype == MZ_BF16) join_t<__bf16>(a, problems, s);
  else join_t<_Float16>(a, problems, s);
}

// bias gradients: dbias[side][f] = sum over the token tiles of col_partial[tile][side][f]; 32 features x 32 tile lanes
template <typename T>
__global__ __launch_bounds__(1024) void bias_grad_kernel(const float* __restrict__ partial, long tiles, long F, T* dbg, T* dbu) {
  __shared__ float red[2][32][33];
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const long f = (long)blockIdx.x * 32 + col;
  float g = 0.f, u = 0.f;
  if (f < F)
    for (long t = lane; t < tiles; t += 32) {
      g += partial[(t * 2 + 0) * F + f];
      u += partial[(t * 2 + 1) * F + f];
    }
  red[0][lane][col] = g;
  red[1][lane][col] = u;
  __syncthreads();
  if (lane >= 2 || f >= F) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) v += red[lane][k][col];
  T* out = lane == 0 ? dbg : dbu;
  if (out) out[f] = (T)v;
}
template <typename T> void bias_grad_t(const float* p, long tiles, long F, void* g, void* u, hipStream_t s) {
  hipLaunchKernelGGL((bias_grad_kernel<T>), dim3((unsigned)((F + 31) / 32)), dim3(1024), 0, s, p, tiles, F,
                     static_cast<T*>(g), static_cast<T*>(u));
}

int64_t tiles(int64_t nr, int64_t nc, int tr, int bc) { return ((nr + tr - 1) / tr) * ((nc + bc - 1) / bc); }

// Tile and split of a product, by its estimated time (microseconds).  A tile's workgroups share a compute unit `at_once`
// at a time; a step of one takes `alone`, and no less than `shared` times the workgroups there; `ends` is what a round
// costs besides its steps (first loads, epilogue), by mode.  A sum cut into parts costs another launch and its partial
// results' way through memory.  Measured per step (64 16-bit or 32 float32 values of k), one workgroup alone / the
// compute unit full, on products of one to 4096 tiles; the estimate is within a fifth of what it was fitted to, and
// choosing by it within a tenth of the best of all choices (18432 x 256 x 1024, dx: 128 x 128 tiles 33 us, 64 x 64 40,
// 256 x 256 48; 1000 x 256 x 1000 float32, dx: 64 x 64 in 4 parts 18 us, 128 x 128 in 16 21, whole 137).
struct TileCost {
  int at_once;
  float alone, shared, ends[3];                    // ends: kForward, kGateGrad, the plain products
};
constexpr TileCost kCost16[3] = {{1, 1.4f, 1.45f, {7.f, 14.f, 8.f}}, {2, .58f, .5f, {3.5f, 6.f, 4.5f}}, {5, .34f, .23f, {2.2f, 4.5f, 2.5f}}};
constexpr TileCost kCost32[3] = {{}, {2, 2.1f, 1.95f, {4.f, 8.f, 5.f}}, {5, .72f, .53f, {2.5f, 4.f, 3.f}}};

struct Split { int tile, splits, steps; };
constexpr int kMaxSplits = 32;

Split pick(int64_t nr, int64_t nc, int64_t steps, int dtype, int mode) {
  const bool pair = mode <= mz_gff::kGateGrad;
  const int problems = mode == mz_gff::kWeightGrad ? 2 : 1;
  const int cus = 256;                             // of an MI355X: the choice, and with it a sum's order, is the same everywhere
  Split best = {2, 1, (int)steps};
  float least = -1.f;
  for (int t = dtype == MZ_F32 ? 1 : 0; t < 3; ++t) {
    const TileCost& c = (dtype == MZ_F32 ? kCost32 : kCost16)[t];
    const int side = mz_gff::tile_side(t);
    const int64_t whole = tiles(nr, nc, pair ? side / 2 : side, side) * problems;
    for (int want = 1; want <= (pair ? 1 : kMaxSplits); want += want < 4 ? 1 : want < 8 ? 2 : want < 16 ? 4 : 8) {
      if (want > 1 && want > steps / 2) break;
      const int64_t per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
      const int64_t share = (whole * splits + cus - 1) / cus, rounds = share / c.at_once, rest = share % c.at_once;
      auto round = [&](int64_t n) {
        const float s = c.shared * n > c.alone ? c.shared * n : c.alone;
        return per * s + c.ends[mode < 2 ? mode : 2];
      };
      float time = rounds * round(c.at_once) + (rest ? round(rest) : 0.f);
      if (splits > 1) time += 3.f + (float)(nr * nc * problems) * splits * 8.f / 8e6f;
      if (least < 0.f || time < least) {
        least = time;
        best = {t, (int)splits, (int)per};
      }
    }
  }
  return best;
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
constexpr int64_t kFew = 64;   // tokens the streaming kernel takes

struct Backward {
  Split dx, dw;
  int gate_tile;
  int64_t dgu_bytes, col_bytes, partial_bytes;
};
Backward plan_backward(const Shape& h) {
  Backward b;
  b.gate_tile = pick(h.F, h.M, h.steps(h.nk_K()), h.dtype, mz_gff::kGateGrad).tile;
  b.dx = pick(h.K, h.M, 2 * h.steps(h.nk_F()), h.dtype, mz_gff::kInputGrad);
  b.dw = pick(h.K, h.F, h.steps(h.nk_M()), h.dtype, mz_gff::kWeightGrad);
  b.dgu_bytes = round_up(h.M * h.Fp * elem_bytes(h.dtype), 256);
  const int side = mz_gff::tile_side(b.gate_tile);
  b.col_bytes = round_up((h.M + side - 1) / side * 2 * h.F * 4, 256);
  const int64_t px = b.dx.splits > 1 ? b.dx.splits * h.M * h.K * 4 : 0, pw = b.dw.splits > 1 ? b.dw.splits * 2 * h.F * h.K * 4 : 0;
  b.partial_bytes = round_up(px > pw ? px : pw, 256);
  return b;
}

int check_shape(const char* who, int64_t M, int64_t K, int64_t F, int32_t dtype, int32_t activation) {
  MZ_REQUIRE(dtype == MZ_F32 || dtype == MZ_BF16 || dtype == MZ_F16, "%s: unknown element type %d", who, dtype);
  MZ_REQUIRE(M > 0 && K > 0 && F > 0 && K <= (1 << 20) && F <= (1 << 20) && M <= (1ll << 40),
             "%s: sizes out of range (M = %lld, K = %lld, F = %lld; K and F up to 2^20)", who, (long long)M, (long long)K,
             (long long)F);
  MZ_REQUIRE(activation >= 0 && activation <= mz_gff::kSigmoid, "%s: unknown activation %d", who, activation);
  return MZ_OK;
}
int check_stride(const char* who, const Shape& h, int64_t ldx) {
  MZ_REQUIRE(ldx >= h.K && ldx * elem_bytes(h.dtype) <= (1 << 22),
             "%s: stride of x out of range (%lld, K = %lld; rows up to 4 MiB apart)", who, (long long)ldx, (long long)h.K);
  return MZ_OK;
}

}  // namespace

extern "C" {

int64_t mz_gated_ff_workspace_bytes(int64_t M, int64_t K, int64_t F, int32_t dtype, int32_t backward) {
  if (check_shape("mz_gated_ff_workspace_bytes", M, K, F, dtype, 0)) return -1;
  if (!backward) return 0;
  const Backward b = plan_backward(make_shape(M, K, F, dtype));
  return 2 * b.dgu_bytes + b.col_bytes + b.partial_bytes;
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
  if (int rc = launch(a, dtype, mz_gff::kForward, pick(F, M, sh.steps(a.nk), dtype, mz_gff::kForward).tile, s)) return rc;
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
  const int64_t need = mz_gated_ff_workspace_bytes(M, K, F, dtype, 1);
  MZ_REQUIRE(workspace && workspace_bytes >= need && (size_t)workspace % 16 == 0,
             "mz_gated_ff_bwd: workspace too small (%lld of %lld bytes) or not 16-byte aligned", (long long)workspace_bytes,
             (long long)need);
  hipStream_t s = mz::as_stream(stream);
  char* dg = static_cast<char*>(workspace);
  char* du = dg + plan.dgu_bytes;
  float* cols = reinterpret_cast<float*>(du + plan.dgu_bytes);
  float* partial = reinterpret_cast<float*>(du + plan.dgu_bytes + plan.col_bytes);
  const bool biases = db_gate || db_up;

  Args a = {};                                     // dg, du
  a.r[0] = w_gate; a.r[1] = w_up;
  a.c[0] = a.c[1] = x;
  a.ldr = K; a.ldc = ldx;
  a.nr = F; a.nc = M; a.nk = sh.nk_K(); a.nk_all = K;
  a.out[0] = dg; a.out[1] = du; a.ldo = sh.Fp;
  a.bias[0] = b_gate; a.bias[1] = b_up;
  a.dh = dh; a.lddh = F;
  a.col_partial = biases ? cols : nullptr;
  a.nr_pad = sh.Fp;
  a.activation = activation;
  a.splits = 1;
  a.steps_per_split = (int)sh.steps(a.nk);
  if (int rc = launch(a, dtype, mz_gff::kGateGrad, plan.gate_tile, s)) return rc;
  if (biases) {
    const int side = mz_gff::tile_side(plan.gate_tile);
    const long n = (long)((M + side - 1) / side);
    if (dtype == MZ_F32) bias_grad_t<float>(cols, n, F, db_gate, db_up, s);
    else if (dtype == MZ_BF16) bias_grad_t<__bf16>(cols, n, F, db_gate, db_up, s);
    else bias_grad_t<_Float16>(cols, n, F, db_gate, db_up, s);
  }
  if (dx) {
    Args p = {};
    p.r[0] = w_gate; p.r[1] = w_up;
    p.c[0] = dg; p.c[1] = du;
    p.ldr = K; p.ldc = sh.Fp;
    p.nr = K; p.nc = M; p.nk = sh.nk_F(); p.nk_all = F;
    p.out[0] = p.out[1] = dx; p.ldo = K;
    p.partial = partial;
    p.splits = plan.dx.splits; p.steps_per_split = plan.dx.steps;
    if (int rc = launch(p, dtype, mz_gff::kInputGrad, plan.dx.tile, s)) return rc;
    if (p.splits > 1) join(p, 1, dtype, s);
  }
  if (dw_gate) {
    Args p = {};
    p.r[0] = p.r[1] = x;
    p.c[0] = dg; p.c[1] = du;
    p.ldr = ldx; p.ldc = sh.Fp;
    p.nr = K; p.nc = F; p.nk = sh.nk_M(); p.nk_all = M;
    p.out[0] = dw_gate; p.out[1] = dw_up; p.ldo = K;
    p.partial = partial;
    p.splits = plan.dw.splits; p.steps_per_split = plan.dw.steps;
    if (int rc = launch(p, dtype, mz_gff::kWeightGrad, plan.dw.tile, s)) return rc;
    if (p.splits > 1) join(p, 2, dtype, s);
  }
  return mz::check_launch("mz_gated_ff_bwd");
}

}  // extern "C"
