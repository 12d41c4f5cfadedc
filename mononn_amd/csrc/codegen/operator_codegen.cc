// Device functions of the operator nodes: a call of the matching template of device/mononn_operators.h with the shapes of
// the custom call as its arguments.
#include <algorithm>
#include <cstdio>
#include <sstream>

#include "codegen/cluster_codegen.h"
#include "common/status.h"

namespace mononn {
namespace codegen {

using hlo::Instr;
using hlo::OperatorConfig;

namespace {

std::string literal(double v, const char* format) {
  char buf[64];
  std::snprintf(buf, sizeof buf, format, v);
  std::string s = buf;
  if (s.find_first_of(".en") == std::string::npos) s += ".0";
  return s;
}
std::string float_literal(double v) { return literal(v, "%.9g") + "f"; }
std::string double_literal(double v) { return literal(v, "%.17g"); }

// elements of one access: the largest power of two up to 16 bytes that divides all of `extents`
int run_length(hlo::DType t, std::initializer_list<int64_t> extents) {
  int v = 16 / hlo::dtype_bytes(t);
  for (int64_t e : extents)
    while (e % v != 0) v /= 2;
  return v;
}

// Heads of a token that one thread takes with the sines it has computed: as many as leave every compute unit `resident`
// threads, at most 8 (what the loads of one thread may hold in registers).
int heads_per_thread(int64_t tokens, int64_t heads, int64_t pieces, int64_t resident) {
  int64_t h = 1;
  while (h < 8 && 2 * h <= heads && tokens * pieces * ((heads + 2 * h - 1) / (2 * h)) >= resident) h *= 2;
  return static_cast<int>(h);
}

bool read_in_kernel(const graph::Program& prog, const Instr* root) {
  for (auto& n : prog.nodes)
    if (std::find(n.inputs.begin(), n.inputs.end(), root) != n.inputs.end()) return true;
  return false;
}

}  // namespace

namespace {
// How matvec_w4 is dealt to the launch: `wk` waves share a tile of 16 weight rows, `sk` workgroups do, a wave reads
// blocks of 128 `p` columns.
struct MatvecPlan {
  int64_t M, N, K, group;
  int64_t wk = 1, sk = 1, p = 1;
  int64_t row_blocks() const { return std::min<int64_t>((M + 15) / 16, 4); }
  int64_t blocks_per_workgroup() const { return ((K + 128 * p - 1) / (128 * p) + sk - 1) / sk; }
  int64_t x_bytes() const { return hlo::matvec_w4_x_bytes(M, blocks_per_workgroup() * p); }
  int64_t lds_bytes(int64_t waves) const { return x_bytes() + (wk > 1 ? waves * row_blocks() * 1024 : 0); }   // and the shares of a tile's waves
  bool fits(int64_t waves) const { return x_bytes() <= hlo::kMatvecW4XBytes && lds_bytes(waves) <= 160 * 1024; }
};
// The plan whose busiest workgroup reads least: weights, its slice of x (16 rows of x on 4096 x 14336 weights: 12.9 us with
// slices of 57 KB of x, 17 with the 115 KB that the weights alone would choose) and its share of the parts (7 rows on
// 5185 x 10880 weights: 12.6 us with 6 slices, 20 with the 43 that would be chosen without).  Among equals larger blocks
// (fewer loads of scales), then fewer slices, then fewer shares (fewer starts of a workgroup's loads).
// What a unit's first loads cost, in 16-byte loads of a workgroup: without it one row on 27648 x 5120 weights takes seven
// rounds of small blocks, 22.6 us instead of 15.8; with 1024 8 rows on 11008 x 4096 take one round, 14.7 instead of 12.3.
constexpr int64_t kUnitStart = 512;
MatvecPlan plan_matvec(const Instr* call, int64_t grid, int64_t waves) {
  const auto &x = call->operands[0]->shape.dims, &w = call->operands[1]->shape.dims, &s = call->operands[2]->shape.dims;
  MatvecPlan best{x[0], w[0], x[1], x[1] / s[1]};
  const bool split = hlo::matvec_w4_in_parts(best.M, best.K);
  const int64_t tiles = (best.N + 15) / 16, passes = (best.M + 16 * best.row_blocks() - 1) / (16 * best.row_blocks());
  const int64_t products = best.M > 4 && best.group >= 128 ? best.row_blocks() : 1;   // a pass of more rows reads more of the LDS for the same weights
  int64_t least = -1;
  // 64 slices at most, unless x is so wide that it takes more: then as few as hold it
  const int64_t columns_at_once = hlo::kMatvecW4XBytes / hlo::matvec_w4_x_bytes(best.M, 1), fewest = split ? ((best.K + 127) / 128 + columns_at_once - 1) / columns_at_once : 1;
  for (int64_t p : {4, 2, 1}) {
    if (p > 1 && best.M > 4 && (best.group >= 128 || p > 2)) continue;   // MatvecW4::kWhole, and the scales of kSwap
    for (int64_t sk = fewest > 64 ? fewest : 1; sk <= (split ? std::max<int64_t>(fewest, 64) : 1); ++sk)
      for (int64_t wk = 1; wk <= waves; wk *= 2) {
        if (waves % wk != 0) break;
        MatvecPlan c = best;
        c.p = p, c.sk = sk, c.wk = wk;
        if (!c.fits(waves)) continue;
        const int64_t at_once = waves / wk, units = (tiles + at_once - 1) / at_once * sk * passes;
        // 16-byte loads of the busiest workgroup: weights and x, and its share of the parts, written and read
        const int64_t parts = split ? sk * best.M * best.N * 8 / 16 / grid : 0;
        const int64_t rounds = (units + grid - 1) / grid, stagings = sk * passes == 1 ? 1 : rounds;
        const int64_t busiest = rounds * ((c.blocks_per_workgroup() + wk - 1) / wk * p * 64 * waves * products + kUnitStart) + stagings * (c.x_bytes() / 16) + parts;
        if (least < 0 || busiest < least) {
          least = busiest;
          best.p = p, best.sk = sk, best.wk = wk;
        }
      }
  }
  MONONN_CHECK(least >= 0, kInternal) << call->hlo_name << ": no arrangement of the 4-bit product fits the LDS";
  return best;
}
}  // namespace

int64_t operator_part_bytes(const Instr* parts, int grid, int waves) {
  const auto& q = parts->operands[0]->shape.dims;
  if (parts->oper.kind == OperatorConfig::kMatvecW4Parts) {
    const MatvecPlan p = plan_matvec(parts, grid, waves);
    return p.sk * p.M * p.N * 4;
  }
  const int64_t group = q[1] / parts->operands[1]->shape.dims[2];
  const int64_t D = q[2], rows = q[0] * group, blocks = std::min<int64_t>((rows + 31) / 32, waves);   // mirrors PagedAttention::kPart
  const int64_t narrow = D / 16 * 256 + 32, wide = blocks * ((D + 31) / 32 * 1024 + 64);   // floats
  return 2 * int64_t(grid) * (rows <= 16 ? narrow : wide) * 4;   // at most 16 query rows in all: no wide item
}

NodeFunction generate_operator(const graph::Program& prog, const graph::Node& node, const LaunchShape& ls, int grid) {
  const Instr* ins = node.members[0];
  const OperatorConfig& c = ins->oper;
  NodeFunction f;
  PointerTable ptrs;
  std::ostringstream body;
  std::vector<std::string> in;
  // storage roots of the operands, as arguments in0 ..
  auto input = [&](size_t i) { return ptrs.input(prog.storage_root(ins->operands[i]), ins->operands[i]->shape.dtype); };
  auto dims = [&](size_t i) -> const std::vector<int64_t>& { return ins->operands[i]->shape.dims; };
  auto ctype = [&](size_t i) { return std::string(hlo::dtype_ctype(ins->operands[i]->shape.dtype)); };
  auto flag = [](bool b) { return b ? "true" : "false"; };
  const int64_t block = ls.block_size, cus = 256;
  auto check_units = [&](int64_t units) {
    MONONN_CHECK(units >= 1 && units < (int64_t(1) << 31), kResourceExhausted) << node.name << " has too many work units";
    f.num_units = units;
  };

  switch (c.kind) {
    case OperatorConfig::kRope: {
      const int64_t T = dims(0)[0], H = dims(0)[1], D = dims(0)[2], R = 2 * dims(2)[0];
      const int vec = run_length(ins->shape.dtype, {R / 2, D, D - R});
      const int64_t pieces = R / 2 / vec + (D - R) / vec;
      const int heads = heads_per_thread(T, H, pieces, cus * block);
      const std::string x = input(0), pos = input(1), freq = input(2), out = ptrs.output(ins);
      body << "mononn_dev::rope_unit<" << ctype(0) << ", " << T << ", " << H << ", " << D << ", " << R << ", " << flag(c.interleaved) << ", " << vec << ", " << heads << ", "
           << flag(read_in_kernel(prog, ins)) << ">(unit, " << x << ", " << pos << ", " << freq << ", " << out << ", " << double_literal(c.amplitude) << ");";
      check_units((T * pieces * ((H + heads - 1) / heads) + block - 1) / block);
      break;
    }
    case OperatorConfig::kKvAppend: {
      const int64_t T = dims(0)[0], H = dims(0)[1], D = dims(0)[2], R = ins->operands.size() == 8 ? 2 * dims(7)[0] : 0;
      const int vec = R > 0 ? run_length(ins->shape.tuple[0].dtype, {R / 2, D, D - R}) : run_length(ins->shape.tuple[0].dtype, {D});
      const int64_t pieces = (R > 0 ? R / 2 / vec : 0) + (D - R) / vec;
      // keys and values side by side: twice the registers of the rotation alone
      const int heads = std::min(4, heads_per_thread(T, H, pieces, cus * block));
      bool coherent = false;
      for (auto* o : node.outputs) coherent = coherent || read_in_kernel(prog, o);
      const std::string k = input(0), v = input(1);
      // the caches are read by nothing else in the kernel, and written at their parameters' addresses
      const std::string kc = ptrs.output(ins->operands[2]), vc = ptrs.output(ins->operands[3]);
      const std::string table = input(4), qs = input(5), cl = input(6), freq = R > 0 ? input(7) : "nullptr";
      body << "mononn_dev::kv_append_unit<" << ctype(0) << ", " << T << ", " << dims(4)[0] << ", " << H << ", " << D << ", " << R << ", " << flag(c.interleaved) << ", " << vec << ", " << heads
           << ", " << dims(2)[1] << ", " << dims(2)[0] << ", " << dims(4)[1] << ", " << flag(coherent) << ">(unit, " << k << ", " << v << ", " << kc << ", " << vc << ", " << table << ", " << qs
           << ", " << cl << ", " << freq << ", " << double_literal(c.amplitude) << ");";
      check_units((T * pieces * ((H + heads - 1) / heads) + block - 1) / block);
      break;
    }
    case OperatorConfig::kPagedAttentionParts:
    case OperatorConfig::kPagedAttention: {
      const bool parts_stage = c.kind == OperatorConfig::kPagedAttentionParts;
      const Instr* parts = parts_stage ? ins : ins->operands[0];
      const Instr* result = parts_stage ? nullptr : ins;
      if (parts_stage)
        for (auto* u : ins->users)
          if (u->oper.kind == OperatorConfig::kPagedAttention) result = u;
      MONONN_CHECK(result != nullptr && parts->oper.kind == OperatorConfig::kPagedAttentionParts, kInternal) << node.name << ": a paged attention without its other stage";
      const auto &q = parts->operands[0]->shape.dims, &kc = parts->operands[1]->shape.dims, &table = parts->operands[3]->shape.dims;
      body << "typedef mononn_dev::PagedAttention<" << hlo::dtype_ctype(result->shape.dtype) << ", " << q[0] << ", " << table[0] << ", " << q[1] << ", " << kc[2] << ", " << q[2] << ", " << kc[1]
           << ", " << kc[0] << ", " << table[1] << ", " << (c.window < table[1] * kc[1] ? c.window : 0) << ", " << grid << ", " << flag(read_in_kernel(prog, result)) << "> Attention; ";
      if (parts_stage) {
        const std::string qp = input(0), kp = input(1), vp = input(2), tp = input(3), sp = input(4), lp = input(5);
        const std::string out = ptrs.output(result), pp = ptrs.output(ins);
        body << "Attention::partial(unit, " << qp << ", " << kp << ", " << vp << ", " << tp << ", " << sp << ", " << lp << ", " << out << ", " << pp << ", " << float_literal(c.scale) << ", smem);";
        // mirrors PagedAttention::lds_bytes
        const int64_t D = q[2], waves = ls.waves(), limit = 160 * 1024;
        const int64_t krow = D * 2 + 16, vrow = (D * 2 + 63) / 128 * 128 + 64, vpn = (D / 16 | 1) * 32, merge = D / 16 * 1024 + 128;
        int64_t nn = waves;
        while (nn > 1 && (nn * 32 * (krow + vpn) > limit || nn * merge > limit)) nn /= 2;
        const int64_t wide = q[0] * (q[1] / kc[2]) <= 16 ? 0 : 64 * (2 * krow + (waves >= 8 && 64 * (2 * krow + 3 * vrow) <= 160 * 1024 ? 3 : 2) * vrow);
        f.smem_bytes = static_cast<int>(std::max({wide, nn * 32 * (krow + vpn), nn * merge}));
        body << " static_assert(Attention::lds_bytes() == " << f.smem_bytes << ", \"LDS\");";
      } else {
        const std::string pp = input(0), sp = input(1), lp = input(2);
        body << "Attention::join(unit, " << pp << ", " << sp << ", " << lp << ", " << ptrs.output(ins) << ", smem);";
        const int64_t tile = q[0] * (q[1] / kc[2]) <= 16 ? 1 : 4;
        f.smem_bytes = static_cast<int>(ls.waves() * (tile * 256 + 128) * 4);
        body << " static_assert(Attention::join_lds_bytes() == " << f.smem_bytes << ", \"LDS\");";
      }
      check_units(grid);
      break;
    }
    case OperatorConfig::kMatvecW4:
    case OperatorConfig::kMatvecW4Parts: {
      const bool parts_stage = c.kind == OperatorConfig::kMatvecW4Parts;
      const Instr* call = parts_stage || ins->operands[0]->oper.kind != OperatorConfig::kMatvecW4Parts ? ins : ins->operands[0];
      const MatvecPlan p = plan_matvec(call, grid, ls.waves());
      const bool zeros = call->operands.size() == 4, join = call != ins;
      body << "typedef mononn_dev::MatvecW4<" << hlo::dtype_ctype(call->operands[0]->shape.dtype) << ", " << p.M << ", " << p.N << ", " << p.K << ", " << p.group << ", " << flag(zeros) << ", "
           << p.wk << ", " << p.sk << ", " << p.p << ", " << flag(!parts_stage && read_in_kernel(prog, ins)) << "> Matvec; ";
      if (join) {
        const std::string pp = input(0);
        body << "Matvec::join(unit, " << pp << ", " << ptrs.output(ins) << ");";
        check_units((p.M * p.N + block - 1) / block);
        break;
      }
      const std::string x = input(0), w = input(1), s = input(2), z = zeros ? input(3) : "nullptr", out = ptrs.output(ins);
      const int64_t at_once = ls.waves() / p.wk, row_blocks = p.row_blocks();
      const int64_t units = ((p.N + 15) / 16 + at_once - 1) / at_once * p.sk * ((p.M + 16 * row_blocks - 1) / (16 * row_blocks));
      check_units(std::min<int64_t>(units, grid));   // a workgroup's units are one unit of the stage: x may stay in its LDS
      body << "Matvec::units<" << f.num_units << ">(unit, " << x << ", " << w << ", " << s << ", " << z << ", " << (parts_stage ? "nullptr, " + out : out + ", nullptr") << ", smem);";
      f.smem_bytes = static_cast<int>(p.lds_bytes(ls.waves()));
      body << " static_assert(Matvec::lds_bytes() == " << f.smem_bytes << " && Matvec::num_units() == " << units << ", \"launch\");";
      break;
    }
    default: MONONN_FAIL(kInternal) << node.name << " is not an operator";
  }
  std::ostringstream os;
  os << "__device__ __forceinline__ void @NAME@(int unit";
  for (auto& e : ptrs.entries) os << ", " << (e.is_output ? "" : "const ") << hlo::dtype_ctype(e.dtype) << "* " << e.name;
  os << ", char* smem) {\n  " << body.str() << "\n}\n";
  f.text = os.str();
  f.pointers = ptrs.entries;
  return f;
}

}  // namespace codegen
}  // namespace mononn
