// Products grouped by expert: checks and the choice of a kernel (gfx950).

#include <string.h>

#include "grouped_gemm.h"

namespace cm {
namespace {

// Whether rows begin on 16 bytes and the axes that are read in pieces of 16 bytes are made of whole ones (offsets within a tile are
// 32-bit, hence the bound on pitches).
bool pieces_whole(const GroupedParams& p, int op, int dtype) {
  const int piece = dtype == CPPMEGA_MI355_E4M3 ? 16 : 8;
  if (((uintptr_t)p.x | (uintptr_t)p.w) & 15) return false;
  if (p.k % piece != 0 || p.x_pitch % piece != 0 || p.x_pitch > (1 << 22) || p.k > (1 << 22)) return false;
  if (op != kRows && p.n % piece != 0) return false;
  return op != kWeightsGrad || (p.w_pitch % piece == 0 && p.w_pitch <= (1 << 22));
}

// How often b x b tiles of a product, `at_once` at a time, are expected to go round (half a tile of rows of each of several experts is padding).
double rounds_of(const GroupedParams& p, int op, int b, int at_once) {
  const double across = ((op == kRows ? p.n : p.k) + b - 1) / b;
  if (op == kWeightsGrad) return (double)p.experts * ((p.n + b - 1) / b) * across / at_once;
  return (p.experts > 1 ? (double)p.rows / b + 0.5 * p.experts : (double)((p.rows + b - 1) / b)) * across / at_once;
}

// 256 x 256 tiles, one to a CU, or 128 x 128, two to a CU: by the rounds that 256 CUs take, a low one's as 0.63 of a high one's (for half the products).
//   Rows: the last round counts less when its tiles are cut.  Measured, us high / low, rows x experts x n x k, bf16: 16384 x 32 x 4096 x 2048 329 / 380,
//   4096 x 1 x 4096 x 4096 120 / 139, 8192 x 64 x 2048 x 2048 185 / 159, 4096 x 16 x 2048 x 2048 64 / 76, 1024 x 1 x 4096 x 4096 60 / 55, 2048 x 8 x 2048 x
//   4096 93 / 73; over 85 such sizes, e4m3 too, the choice loses 0.5 % to the better one.
//   Weights: half a round is idle at the end.  512 x 16 x 4096 x 2048 75 / 96, 8192 x 1 x 4096 x 4096 216 / 254, 1024 x 1 x 2048 x 1024 29 / 16, 2048 x 8 x 1000 x
//   1544 31 / 20; the worst of 56 sizes 12 % (512 x 32 x 2048 x 2048 92 / 83).
bool high_tiles(const GroupedParams& p, int op) {
  auto rounds = [&](int b, int at_once, double quarter, double half) {
    const double x = rounds_of(p, op, b, at_once), whole = (double)(long long)x, last = x - whole;
    if (op == kWeightsGrad) return x > 0.5 ? x + 0.5 : 1.0;
    return whole + (last == 0.0 ? 0.0 : last <= 0.25 ? quarter : last <= 0.5 ? half : 1.0);
  };
  return rounds(256, 256, 0.5, 0.67) <= 0.63 * rounds(128, 512, 0.62, 0.62);
}

// Both gradients in one launch: whole rounds of all tiles, the rows' first and uncut.  Measured as above: 8192 x 16 x 4096 x 2048 327 / 389, 512 x 16 x 4096 x
// 2048 126 / 162, 512 x 1 x 4096 x 4096 86 / 49, 2048 x 8 x 2048 x 4096 119 / 135, 2048 x 1 x 4096 x 4096 122 / 145 (where the rule takes the low ones).
bool high_grads(const GroupedParams& rows, const GroupedParams& weights) {
  auto rounds = [&](int b, int at_once) {
    const double x = rounds_of(rows, kRowsGrad, b, at_once) + rounds_of(weights, kWeightsGrad, b, at_once), whole = (double)(long long)x;
    return x > whole ? whole + 1.0 : whole;
  };
  return rounds(256, 256) <= 0.63 * rounds(128, 512);
}

// What a call runs: nothing, or one of the kernels.
enum Kind { kNothing, kGeneral, kStream, kTile };
struct Plan {
  GroupedParams p;
  Kind kind;
  bool high, gated;
};

int plan_of(const char* call, const cppmega_mi355_grouped_gemm_args_t& a, Plan& to) {
  to.kind = kNothing;
  to.gated = false;
  if (a.op < kRows || a.op > kWeightsGrad) return fail(CPPMEGA_MI355_ERR_SHAPE, "%s: unknown op %d", call, a.op);
  if (a.rows < 0 || a.rows > 0x1fffffffll || a.experts < 1 || a.n < 1 || a.k < 1)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "%s: rows=%lld experts=%d k=%d, weights of %d rows", call, (long long)a.rows, a.experts, a.k, a.n);
  // (columns and contraction are counted in 32 bits, a tile past the end)
  if (a.n > CPPMEGA_MI355_GROUPED_MAX_SIZE || a.k > CPPMEGA_MI355_GROUPED_MAX_SIZE)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "%s: k=%d, weights of %d rows; at most 2^30 are served", call, a.k, a.n);
  if (a.experts > kMaxExperts) return fail(CPPMEGA_MI355_ERR_UNSUPPORTED, "%s: %d experts, at most %d are served", call, a.experts, kMaxExperts);
  const bool fp8 = a.x_dtype == CPPMEGA_MI355_E4M3;
  if (!fp8 && a.x_dtype != CPPMEGA_MI355_F16 && a.x_dtype != CPPMEGA_MI355_BF16)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "%s: operands of dtype %d are not float16 / bfloat16 / e4m3", call, a.x_dtype);
  if (fp8 && a.op != kRows) return fail(CPPMEGA_MI355_ERR_DTYPE, "%s: gradients of e4m3 operands are not served", call);
  if (fp8 ? a.y_dtype != CPPMEGA_MI355_F32 && a.y_dtype != CPPMEGA_MI355_F16 && a.y_dtype != CPPMEGA_MI355_BF16
          : a.y_dtype != CPPMEGA_MI355_F32 && a.y_dtype != a.x_dtype)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "%s: a result of dtype %d from operands of dtype %d", call, a.y_dtype, a.x_dtype);
  if (a.offsets_dtype != CPPMEGA_MI355_I32 && a.offsets_dtype != CPPMEGA_MI355_I64)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "%s: offsets must be int32 or int64", call);
  if (fp8 && a.x_scale_block != 0 && a.x_scale_block != 128)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "%s: x_scale_block must be 0 (per row) or 128, got %d", call, a.x_scale_block);
  if (a.rows == 0 && a.op != kWeightsGrad) return 0;
  if (!a.y || (!a.offsets && a.experts != 1) || (a.rows > 0 && (!a.x || !a.w)) || (fp8 && (!a.x_scale || !a.w_scale)))
    return fail(CPPMEGA_MI355_ERR_NULL, "%s: x / w / y / offsets / scales is NULL", call);
  GroupedParams& p = to.p;
  memset(&p, 0, sizeof(p));
  p.x = a.x; p.w = a.w; p.y = a.y; p.offsets = a.offsets; p.x_scale = a.x_scale; p.w_scale = a.w_scale;
  p.rows = a.rows; p.x_pitch = a.x_pitch; p.w_pitch = a.w_pitch; p.y_pitch = a.y_pitch;
  p.experts = a.experts; p.n = a.n; p.k = a.k;
  p.y_dtype = a.y_dtype; p.offsets64 = a.offsets_dtype == CPPMEGA_MI355_I64; p.x_scale_block = a.x_scale_block; p.zero_tail = a.zero_tail;
  to.kind = kGeneral;
  if (pieces_whole(p, a.op, a.x_dtype)) {
    // Few rows to an expert: the kernel that streams the weights, 16 rows at a time.  Measured against tiles, us, rows to an expert on average (drawn
    // at random): 64 experts of 2048 x 2048, bf16 8 96 / 129, 14 109 / 130, 20 143 / 131; of 4096 x 2048 8 184 / 185, 14 209 / 187, 20 275 / 189; e4m3 8
    // 48 / 49 and 97 / 108, 12 51 / 49 and 104 / 109, 20 77 / 50 and 151 / 121.  float16 and float32 results of e4m3
    // operands have the general kernel instead of tiles: 20 78 / 136, 48 145 / 149.  The offsets stay on the device, so the rule knows the mean only:
    // with all rows in one expert of 64 its weights are read once for every 16 of them (4096 x 2048 bf16, 890 rows: 128 us, where the tiles take 30 and an
    // even call 186), with half of them there the call takes 239.
    const bool exact = fp8 && a.y_dtype != CPPMEGA_MI355_BF16;
    if (a.op == kRows && a.rows < (exact ? 48ll : fp8 ? 12ll : 14ll) * a.experts) {
      to.kind = kStream;
    } else if (!exact) {                                         // (the tiles' matrix instruction for e4m3 drops low products)
      to.kind = kTile;
      to.high = high_tiles(p, a.op);
    }
  }
  return 0;
}

int check(const char* call, const Plan& plan, int op) {
  if (plan.kind == kTile) return grouped_tile_check(call, plan.p, op, plan.high, plan.gated);
  if (plan.kind == kStream) return grouped_stream_check(call, plan.p, plan.gated);
  return plan.kind == kGeneral ? grouped_general_check(call, plan.p, op, plan.gated) : 0;
}

int launch(const char* call, const Plan& plan, int op, int dtype, hipStream_t stream) {
  if (int rc = check(call, plan, op)) return rc;
  if (plan.kind == kTile) return grouped_tile_launch(plan.p, op, dtype, plan.high, plan.gated, stream);
  if (plan.kind == kStream) return grouped_stream_launch(plan.p, dtype, plan.gated, stream);
  return plan.kind == kGeneral ? grouped_general_launch(plan.p, op, dtype, plan.gated, stream) : 0;
}

// The gradients that are wanted, and whether one launch makes both; everything that may refuse either of them is asked here.
int plan_grads(const char* call, const cppmega_mi355_grouped_gemm_args_t& rows, const cppmega_mi355_grouped_gemm_args_t& weights, bool need_rows, bool need_weights, Plan& r, Plan& w,
               bool& together) {
  if (rows.op != kRowsGrad || weights.op != kWeightsGrad)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "%s: ops %d and %d are not the rows' and the weights' gradient", call, rows.op, weights.op);
  int rc = need_rows ? plan_of(call, rows, r) : 0;
  if (!rc && need_weights) rc = plan_of(call, weights, w);
  if (rc) return rc;
  together = need_rows && need_weights && r.kind == kTile && w.kind == kTile && rows.x_dtype == weights.x_dtype;
  if (together) {
    r.high = w.high = high_grads(r.p, w.p);
    return grouped_tile_grads_check(call, r.p, w.p, r.high);
  }
  rc = need_rows ? check(call, r, kRowsGrad) : 0;
  return !rc && need_weights ? check(call, w, kWeightsGrad) : rc;
}

}  // namespace

// (`call`: the entry point that a refusal names)
int grouped_gemm_launch_as(const char* call, const cppmega_mi355_grouped_gemm_args_t& a, hipStream_t stream) {
  Plan plan;
  if (int rc = plan_of(call, a, plan)) return rc;
  return launch(call, plan, a.op, a.x_dtype, stream);
}
int grouped_gemm_launch(const cppmega_mi355_grouped_gemm_args_t& a, hipStream_t stream) { return grouped_gemm_launch_as("grouped_gemm", a, stream); }

int grouped_gemm_bwd_launch_as(const char* call, const cppmega_mi355_grouped_gemm_args_t& rows, const cppmega_mi355_grouped_gemm_args_t& weights, hipStream_t stream) {
  Plan r, w;
  bool together;
  if (int rc = plan_grads(call, rows, weights, true, true, r, w, together)) return rc;
  if (together) return grouped_tile_grads_launch(r.p, w.p, rows.x_dtype, r.high, stream);
  const int rc = launch(call, r, kRowsGrad, rows.x_dtype, stream);
  return rc ? rc : launch(call, w, kWeightsGrad, weights.x_dtype, stream);
}
int grouped_gemm_bwd_launch(const cppmega_mi355_grouped_gemm_args_t& rows, const cppmega_mi355_grouped_gemm_args_t& weights, hipStream_t stream) {
  return grouped_gemm_bwd_launch_as("grouped_gemm_bwd", rows, weights, stream);
}

// Whether the gradients that are wanted would be launched, with the reason if not.
int grouped_gemm_check(const char* call, const cppmega_mi355_grouped_gemm_args_t& rows, const cppmega_mi355_grouped_gemm_args_t& weights, bool need_rows, bool need_weights) {
  Plan r, w;
  bool together;
  return plan_grads(call, rows, weights, need_rows, need_weights, r, w, together);
}

// The gated block is a product of rows with 2 n rows of a weight, whose kernels pair them off; the same rules choose among them.
int gated_gemm_launch(const cppmega_mi355_gated_gemm_args_t& a, hipStream_t stream) {
  if (a.activation != CPPMEGA_MI355_GATE_SILU && a.activation != CPPMEGA_MI355_GATE_GELU_TANH)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "gated_gemm: unknown activation %d", a.activation);
  if (a.n < 1 || a.n > CPPMEGA_MI355_GATED_MAX_OUTPUTS) return fail(CPPMEGA_MI355_ERR_SHAPE, "gated_gemm: n=%d, 1 to 2^29 are served", a.n);
  if (a.pre && a.x_dtype == CPPMEGA_MI355_E4M3) return fail(CPPMEGA_MI355_ERR_DTYPE, "gated_gemm: the products of e4m3 operands are not kept");
  if (a.pre && a.pre_dtype != a.x_dtype && a.pre_dtype != CPPMEGA_MI355_F32)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "gated_gemm: pre of dtype %d from operands of dtype %d", a.pre_dtype, a.x_dtype);
  cppmega_mi355_grouped_gemm_args_t g;
  memset(&g, 0, sizeof(g));
  g.op = kRows;
  g.x = a.x; g.w = a.w; g.y = a.y; g.offsets = a.offsets; g.x_scale = a.x_scale; g.w_scale = a.w_scale;
  g.x_dtype = a.x_dtype; g.y_dtype = a.y_dtype; g.offsets_dtype = a.offsets_dtype; g.x_scale_block = a.x_scale_block;
  g.rows = a.rows; g.x_pitch = a.x_pitch; g.y_pitch = a.y_pitch;
  g.experts = a.experts; g.n = 2 * a.n; g.k = a.k; g.zero_tail = a.zero_tail;
  Plan plan;
  if (int rc = plan_of("gated_gemm", g, plan)) return rc;
  plan.gated = true;
  plan.p.n = a.n;
  plan.p.activation = a.activation;
  plan.p.pre = a.pre; plan.p.pre_dtype = a.pre_dtype; plan.p.pre_pitch = a.pre_pitch;
  // Few tiles leave most CUs without work, and each goes through the whole contraction: the kernel that streams the weights has more
  // workgroups, and passes them once for 16 rows.  Measured, us stream / tiles, rows x n x k of one expert: bf16 64 x 2048 x 4096 25 / 33, 128 x 2048 x 4096
  // 39 / 33, 16 x 8192 x 2048 15 / 22, 32 x 8192 x 2048 24 / 22, 64 x 1024 x 7168 22 / 59, 128 x 1024 x 1024 8.5 / 11, 200 x 512 x 2048 14 / 16; e4m3 64 x 2048 x
  // 4096 16 / 19, 128 x 2048 x 4096 24 / 19; 512 x 8 experts x 512 x 2048 31 / 21.
  const double passes = a.experts > 1 ? a.rows / 16.0 + 0.5 * a.experts : (double)((a.rows + 15) / 16);
  if (plan.kind == kTile && passes * a.n <= 8192.0) plan.kind = kStream;
  return launch("gated_gemm", plan, kRows, a.x_dtype, stream);
}

}  // namespace cm
