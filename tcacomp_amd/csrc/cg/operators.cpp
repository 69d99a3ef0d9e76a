// operators.cpp — see operators.h. The kernels are templates of
// tca/hip/norm.h and tca/hip/product.h; what is emitted here is their
// instances for one set of attributes and the plan that picks among them.
#include "operators.h"

#include <map>
#include <set>
#include <sstream>
#include <vector>

namespace tca {
namespace cg {

namespace {

struct Spec {
  const char* name;
  std::vector<std::string> elems;
  bool weight, nobias, bias, stats, residual, save, act;
  std::vector<std::string> more;  // flags of its own
};

const std::vector<Spec>& Specs() {
  static const std::vector<Spec> specs = {
      {"layer_norm", {"f32", "bf16", "f16"}, true, true, false, true, false, false, false, {}},
      {"layer_norm_backward", {"f32", "bf16", "f16"}, true, true, false, false, true, false, false, {}},
      {"linear", {"bf16", "f16"}, false, false, true, false, true, true, true, {}},
      {"linear_backward", {"bf16", "f16"}, false, false, true, false, false, false, true, {}},
      {"gated", {"bf16", "f16"}, false, false, true, false, false, true, true, {}},
      {"gated_backward", {"bf16", "f16"}, false, false, true, false, false, false, true, {}},
      {"page_table", {}, false, false, false, false, false, false, false, {}},
      {"rotary", {"f32", "bf16", "f16"}, false, false, false, false, false, false, false, {"interleaved", "inverse"}},
      {"rotary_cache", {"f32", "bf16", "f16"}, false, false, false, false, false, false, false, {"interleaved"}},
      {"paged_attention", {"bf16", "f16"}, false, false, false, true, false, false, false, {"window"}},
  };
  return specs;
}

const std::vector<std::string>& Acts() {
  static const std::vector<std::string> acts = {"none", "relu", "silu", "gelu", "gelu_tanh"};
  return acts;
}

std::vector<std::string> Flags(const Spec& s) {
  std::vector<std::string> f;
  if (s.nobias) f.push_back("nobias");
  if (s.bias) f.push_back("bias");
  if (s.stats) f.push_back("stats");
  if (s.residual) f.push_back("residual");
  if (s.save) f.push_back("save");
  f.insert(f.end(), s.more.begin(), s.more.end());
  return f;
}

std::string Join(const std::vector<std::string>& v, const char* sep) {
  std::string s;
  for (const auto& x : v) s += (s.empty() ? "" : sep) + x;
  return s;
}

std::string Usage(const Spec& s) {
  std::string u = s.elems.empty() ? "no attributes" : "elem=" + Join(s.elems, "|");
  if (s.weight) u += " [weight=f32]";
  if (s.act) u += " [act=" + Join(Acts(), "|") + "]";
  for (const auto& f : Flags(s)) u += " [" + f + "]";
  return u;
}

bool Has(const std::vector<std::string>& v, const std::string& x) {
  for (const auto& y : v)
    if (x == y) return true;
  return false;
}

// The attributes of one program.
struct Attrs {
  std::string elem, weight, act = "none";
  std::set<std::string> flags;
  bool Flag(const char* f) const { return flags.count(f) != 0; }
};

bool ParseAttrs(const Spec& s, const std::string& text, Attrs* a, std::string* err) {
  const std::string takes = std::string("; ") + s.name + " takes " + Usage(s);
  if (std::string(s.name).rfind("gated", 0) == 0) a->act = "silu";
  std::set<std::string> seen;
  std::istringstream in(text);
  for (std::string w; in >> w;) {
    const size_t eq = w.find('=');
    const std::string key = w.substr(0, eq), value = eq == std::string::npos ? "" : w.substr(eq + 1);
    if (!seen.insert(key).second) {
      *err = "operator " + std::string(s.name) + ": attribute " + key + " is given twice";
      return false;
    }
    bool ok = true;
    if (eq == std::string::npos) {
      ok = Has(Flags(s), key);
      if (ok) a->flags.insert(key);
    } else if (key == "elem") {
      ok = Has(s.elems, value);
      a->elem = value;
    } else if (key == "weight") {
      ok = s.weight && value == "f32";
      a->weight = value;
    } else if (key == "act") {
      ok = s.act && Has(Acts(), value);
      a->act = value;
    } else {
      ok = false;
    }
    if (!ok) {
      *err = "operator " + std::string(s.name) + ": unsupported attribute " + w + takes;
      return false;
    }
  }
  if (a->elem.empty() && !s.elems.empty()) {
    *err = "operator " + std::string(s.name) + ": no elem" + takes;
    return false;
  }
  if (a->weight.empty()) a->weight = a->elem;
  return true;
}

std::string ElemType(const std::string& e) { return e == "f32" ? "float" : e == "i32" ? "int32_t" : e == "u32" ? "uint32_t" : e == "bf16" ? "__bf16" : "_Float16"; }
std::string Bool(bool b) { return b ? "true" : "false"; }

// The source and plan of a program as they grow.
class Writer {
 public:
  explicit Writer(const std::string& program) : program_(program) {}

  void Dim(const std::string& name, uint64_t extent = 0) { dims_ << "dim " << name << " " << extent << "\n"; }
  // `dims`: names separated by spaces.
  void Tensor(const std::string& name, const std::string& elem, const char* role, const std::string& dims) {
    int rank = 0;
    std::istringstream in(dims);
    for (std::string d; in >> d;) ++rank;
    tensors_ << "tensor " << name << " " << elem << " " << role << " " << rank << " " << dims << "\n";
    types_[name] = std::make_pair(ElemType(elem), std::string(role) == "in");
  }
  // A tensor of 4-byte values that kernels read and write one by one: it may start at any of them.
  void List(const std::string& name, const std::string& elem, const char* role, const std::string& dims) {
    Tensor(name, elem, role, dims);
    tensors_ << "align " << name << " 4\n";
  }
  bool Has(const std::string& tensor) const { return types_.count(tensor) != 0; }
  void Scalar(const std::string& name) {
    scalars_ << "scalar " << name << " f32\n";
    scalar_names_.insert(name);
  }
  // What the dims have to satisfy (the plan's require record).
  void Require(const std::string& record) { requires_ << "require " << record << "\n"; }
  void Header(const std::string& h) { headers_ << "#include \"" << h << "\"\n"; }
  void Comment(const std::string& c) { body_ << "// " << c << "\n"; }

  struct Kernel {
    std::string suffix, params, body, grid, detail;  // params: tensor, dim and scalar names; grid: terms
    uint32_t block = 256;
    uint32_t waves = 0;  // on a SIMD, that its registers have to leave room for
    std::vector<std::string> records;  // when, unless, split, scratch
    // Functions that stand in for it: their suffix, body and what they are, and
    // the plan's bounds (after "form <symbol>"); one may be listed again with others.
    struct Form {
      std::string suffix, body, detail, bounds;
    };
    std::vector<Form> forms;
  };
  void Add(const Kernel& k) {
    const std::string symbol = "tca_" + program_ + k.suffix;
    std::istringstream in(k.params);
    std::string sig, args;
    for (std::string p; in >> p;) {
      sig += sig.empty() ? "" : ", ";
      const auto t = types_.find(p);
      if (t != types_.end()) {
        sig += (t->second.second ? "const " : "") + t->second.first + "* " + p;
        args += "arg ptr " + p + "\n";
      } else if (scalar_names_.count(p) != 0) {
        sig += "float " + p;
        args += "arg scalar " + p + "\n";
      } else {
        sig += "uint32_t " + p;
        args += "arg dim " + p + "\n";
      }
    }
    auto function = [&](const std::string& name, const std::string& detail, const std::string& body) {
      body_ << "// " << detail << "\nextern \"C\" __global__ void __launch_bounds__(" << k.block
            << (k.waves != 0u ? ", " + std::to_string(k.waves) : "") << ") " << name << "("
            << sig << ") {\n" << body << "}\n\n";
    };
    function(symbol, k.detail, k.body);
    std::set<std::string> written;
    for (const auto& f : k.forms)
      if (written.insert(f.suffix).second) function("tca_" + program_ + f.suffix, f.detail, f.body);
    int terms = 0;
    std::istringstream g(k.grid);
    for (std::string t; g >> t;) ++terms;
    kernels_ << "kernel " << symbol << " " << k.block << " 0 " << terms << " " << k.grid << "\n" << args;
    for (const auto& f : k.forms) kernels_ << "form tca_" << program_ << f.suffix << " " << f.bounds << "\n";
    for (const auto& r : k.records) kernels_ << r << "\n";
    report_ << symbol << " operator chains= " << k.detail << "\n";
    KernelInfo info;
    info.symbol = symbol;
    info.detail = k.detail;
    infos_.push_back(info);
  }

  void Finish(const std::string& target, Result* out) const {
    out->source = "// " + program_ + " for " + target + "\n#include <hip/hip_runtime.h>\n#include <stdint.h>\n\n" +
                  headers_.str() + "\n" + body_.str();
    out->plan = "tca-plan 1\nprogram " + program_ + "\n" + dims_.str() + tensors_.str() + scalars_.str() +
                requires_.str() + kernels_.str() + "end\n";
    out->hipcc = DeviceFlags(target);
    out->kernels = infos_;
    out->report = report_.str();
  }

 private:
  std::string program_;
  std::ostringstream dims_, tensors_, scalars_, requires_, headers_, body_, kernels_, report_;
  std::set<std::string> scalar_names_;
  std::map<std::string, std::pair<std::string, bool>> types_;  // tensor -> element type, const
  std::vector<KernelInfo> infos_;
};

std::string When(const std::string& dims, uint64_t lo, uint64_t hi, uint64_t mod = 1) {
  return "when " + dims + " " + std::to_string(lo) + " " + std::to_string(hi) + " " + std::to_string(mod) + " 0";
}
constexpr uint64_t kMost = 4294967295ull;
// What a kernel writes of local `tensor`, as grid terms.
std::string Scratch(const std::string& tensor, const std::string& terms) {
  int n = 0;
  std::istringstream in(terms);
  for (std::string t; in >> t;) ++n;
  return "scratch " + tensor + " " + std::to_string(n) + " " + terms;
}

// ------------------------------------------------------------- layer norm

// The lanes and vectors that hold a row, by its length in 16-byte vectors.
constexpr uint32_t kLanes = 256 * 2048;  // of the card
struct RowForm {
  uint32_t lanes, vectors;
  uint32_t Span() const { return lanes * vectors; }
};

void EmitLayerNorm(const Attrs& a, Writer* w) {
  const bool bias = !a.Flag("nobias"), stats = a.Flag("stats");
  w->Header("tca/hip/norm.h");
  w->Dim("R");
  w->Dim("C");
  w->Tensor("x", a.elem, "in", "R C");
  w->Tensor("gamma", a.weight, "in", "C");
  if (bias) w->Tensor("beta", a.weight, "in", "C");
  w->Tensor("y", a.elem, "out", "R C");
  if (stats) {
    w->Tensor("mean", "f32", "out", "R");
    w->Tensor("rstd", "f32", "out", "R");
  }
  w->Scalar("eps");
  const std::string params = std::string("x gamma ") + (bias ? "beta " : "") + "y " + (stats ? "mean rstd " : "") + "R C eps";
  const std::string T = ElemType(a.elem), W = ElemType(a.weight);
  const std::string args = std::string("(x, gamma, ") + (bias ? "beta" : "(const " + W + "*)nullptr") + ", y, " +
                           (stats ? "mean, rstd" : "(float*)nullptr, (float*)nullptr") + ", R, C, eps);\n";
  const std::string tail = ", " + Bool(bias) + ", " + Bool(stats) + ">" + args;
  const uint32_t E = a.elem == "f32" ? 4u : 8u;
  uint64_t from = 0;
  for (const RowForm& f : {RowForm{16, 1}, RowForm{64, 1}, RowForm{64, 2}, RowForm{64, 4}, RowForm{256, 2},
                           RowForm{256, 4}, RowForm{1024, 2}, RowForm{1024, 4}}) {
    // 16 waves have 128 registers each: 16-bit rows with f32 weights would spill.
    if (f.Span() == 4096u && a.elem != a.weight) continue;
    const uint64_t to = static_cast<uint64_t>(f.Span()) * E;
    const uint32_t block = f.lanes < 256u ? 256u : f.lanes;
    const std::string g = std::to_string(f.lanes), v = std::to_string(f.vectors);
    Writer::Kernel k;
    k.suffix = "_" + g + "x" + v;
    k.params = params;
    k.block = block;
    k.body = "  tca::hip::norm_rows<" + T + ", " + W + ", " + g + ", " + v + tail;
    // At most 2048 lanes a CU, eight waves a SIMD. The narrow forms fit so; 64x4 (93
    // VGPRs in f32, 141 in f16) has five and three waves resident and 256x4 (115,
    // 188) four and two: their workgroups come in two to four rounds.
    k.grid = "R/" + std::to_string(block / f.lanes) + ":" + std::to_string(kLanes / block);
    k.records = {When("C", from, to)};
    k.detail = "rows of " + std::to_string(from) + " to " + std::to_string(to) + " in registers, " + g + " lanes of " + v + " vectors";
    w->Add(k);
    from = to + 1;
  }
  Writer::Kernel k;
  k.suffix = "_long";
  k.params = params;
  k.block = 1024;
  k.body = "  tca::hip::norm_long<" + T + ", " + W + tail;
  k.grid = "R/1";
  k.records = {When("C", from, kMost)};
  k.detail = "rows from " + std::to_string(from) + " on, read twice, 1024 lanes";
  w->Add(k);
}

void EmitLayerNormBackward(const Attrs& a, Writer* w) {
  const bool bias = !a.Flag("nobias"), res = a.Flag("residual");
  w->Header("tca/hip/norm.h");
  w->Dim("R");
  w->Dim("C");
  // Partial rows of the weights' gradients: at most 16 MiB of them for rows
  // in registers (8192 values by two gradients).
  const uint32_t kParts = 256, kLongParts = 32;
  w->Dim("parts", kParts);
  w->Dim("long_parts", kLongParts);
  w->Dim("grads", bias ? 2 : 1);
  w->Tensor("dy", a.elem, "in", "R C");
  w->Tensor("x", a.elem, "in", "R C");
  w->Tensor("gamma", a.weight, "in", "C");
  w->Tensor("mean", "f32", "in", "R");
  w->Tensor("rstd", "f32", "in", "R");
  if (res) w->Tensor("dres", a.elem, "in", "R C");
  w->Tensor("dx", a.elem, "out", "R C");
  w->Tensor("dgamma", a.weight, "out", "C");
  if (bias) w->Tensor("dbeta", a.weight, "out", "C");
  w->Tensor("part", "f32", "local", "parts grads C");
  w->Tensor("long_part", "f32", "local", "long_parts grads C");
  const std::string T = ElemType(a.elem), W = ElemType(a.weight), none = "(const " + T + "*)nullptr";
  const std::string ins = std::string("dy x gamma mean rstd ") + (res ? "dres " : "") + "dx ";
  const std::string args = "(dy, x, gamma, mean, rstd, " + (res ? "dres" : none) + ", dx, ";
  const uint32_t E = a.elem == "f32" ? 4u : 8u;
  uint64_t from = 0;
  auto scratch = [&](const std::string& part, uint32_t groups, uint32_t most) {
    return Scratch(part, "R/" + std::to_string(groups) + ":" + std::to_string(most) + " C/1" + (bias ? " 2/1" : ""));
  };
  auto join = [&](const std::string& suffix, const std::string& part, uint32_t groups, uint32_t most, uint64_t lo, uint64_t hi) {
    Writer::Kernel j;
    j.suffix = suffix;
    j.params = part + " dgamma " + (bias ? "dbeta " : "") + "R C";
    j.body = "  tca::hip::join_partials<" + W + ">(" + part + ", dgamma, " + (bias ? "dbeta" : "(" + W + "*)nullptr") + ", " +
             (bias ? "2u" : "1u") + ", C, tca::hip::partial_rows(R, " + std::to_string(groups) + "u, " + std::to_string(most) + "u));\n";
    j.block = 1024;
    j.grid = std::string("C/32") + (bias ? " 2/1" : "");
    j.records = {When("C", lo, hi)};
    j.detail = "the weights' gradients from the partial rows of " + std::to_string(groups) + " at a time";
    w->Add(j);
  };
  for (const RowForm& f : {RowForm{16, 1}, RowForm{64, 1}, RowForm{64, 2}, RowForm{256, 1}, RowForm{256, 2},
                           RowForm{512, 2}, RowForm{512, 4}}) {
    if (f.vectors == 4u && E == 8u) continue;  // two rows, their sums and the gradients' do not fit 256 registers
    const uint64_t to = static_cast<uint64_t>(f.Span()) * E;
    const uint32_t groups = 512u / f.lanes;
    const std::string g = std::to_string(f.lanes), v = std::to_string(f.vectors);
    Writer::Kernel k;
    k.suffix = "_" + g + "x" + v;
    k.params = ins + "part R C";
    k.block = 512;
    k.body = "  tca::hip::norm_backward_rows<" + T + ", " + W + ", " + g + ", " + v + ", " + Bool(bias) + ", " + Bool(res) +
             ">" + args + "part, R, C);\n";
    k.grid = "R/" + std::to_string(groups) + ":" + std::to_string(kParts);
    k.records = {When("C", from, to), scratch("part", groups, kParts)};
    k.detail = "rows of " + std::to_string(from) + " to " + std::to_string(to) + " in registers, " + g + " lanes of " + v +
               " vectors, partial weight gradients";
    w->Add(k);
    join(k.suffix + "_join", "part", groups, kParts, from, to);
    from = to + 1;
  }
  Writer::Kernel k;
  k.suffix = "_long";
  k.params = ins + "R C";
  k.block = 1024;
  k.body = "  tca::hip::norm_backward_long<" + T + ", " + W + ", " + Bool(res) + ">" + args + "R, C);\n";
  k.grid = "R/1";
  k.records = {When("C", from, kMost)};
  k.detail = "rows from " + std::to_string(from) + " on, read twice, 1024 lanes";
  w->Add(k);
  Writer::Kernel c;
  c.suffix = "_columns";
  c.params = "dy x mean rstd long_part R C";
  const std::string parts = "tca::hip::partial_rows(R, 64u, " + std::to_string(kLongParts) + "u)";
  c.body = "  tca::hip::norm_backward_columns<" + T + ", " + Bool(bias) + ">(dy, x, mean, rstd, long_part, R, C, " + parts + ");\n";
  c.grid = "C/" + std::to_string(64u * E) + " R/64:" + std::to_string(kLongParts);
  c.records = {When("C", from, kMost), scratch("long_part", 64, kLongParts)};
  c.detail = "partial weight gradients of rows from " + std::to_string(from) + " on, by columns";
  w->Add(c);
  join("_long_join", "long_part", 64, kLongParts, from, kMost);
}

// --------------------------------------------------------------- products

int ActCode(const std::string& act) {
  for (size_t i = 0; i < Acts().size(); ++i)
    if (Acts()[i] == act) return static_cast<int>(i);
  return 0;
}

// One product of a program: its operands and epilogue as source text.
struct Product {
  std::string suffix, what;
  std::string M, N, K;                // dims: rows, columns and reduction
  std::string A[2], B[2][2];          // [segment], [half][segment]
  bool a_rc = false, b_rc = false, pair = false;
  int segs = 1;
  std::string params;                 // operands, epilogue tensors and dims
  std::string epi;                    // an expression of the epilogue's type
};

// Rows of a forward product that product_few takes.
constexpr uint32_t kFewRows = 64;
// Workgroups that products of few tiles are split into, by k: as many as CUs.
constexpr uint32_t kCUs = 256;
// Planes of at most so many results may be split (64 tiles of 128x128: into four and
// more; two parts pay for the sum of their halves more than they save: dx of 2048 x
// 1024 x 4096, 128 tiles, 25 and 5 us in two parts, 25 in one of half the tile).
constexpr uint64_t kSplitPlane = 1ull << 20;

void EmitProduct(const Attrs& a, const Product& p, Writer* w) {
  std::ostringstream ops;
  ops << "  tca::hip::Operands<" << p.segs << "> p;\n";
  for (int s = 0; s < p.segs; ++s) {
    ops << "  p.a[" << s << "] = reinterpret_cast<const uint16_t*>(" << p.A[s] << ");\n";
    for (int h = 0; h < 2; ++h)
      ops << "  p.b[" << h << "][" << s << "] = reinterpret_cast<const uint16_t*>(" << p.B[p.pair ? h : 0][s] << ");\n";
  }
  ops << "  p.M = " << p.M << ";\n  p.N = " << p.N << ";\n  p.K = " << p.K << ";\n  const auto epi = " << p.epi << ";\n";
  const std::string f16 = Bool(a.elem == "f16"), pair = Bool(p.pair);
  const std::string targs = f16 + ", " + Bool(p.a_rc) + ", " + Bool(p.b_rc) + ", " + pair + ", " + std::to_string(p.segs);
  const std::string plane = p.M + "*" + p.N, part = "part";
  const std::string sums = Scratch(part, plane + "/1" + (p.pair ? " 2/1" : ""));  // of each of P parts
  // Tiles of rows x cols (of a pair: cols / 2 of each product) as grid terms, and counted on the device.
  auto tiles = [&](uint32_t rows, uint32_t cols) {
    return p.M + "/" + std::to_string(rows) + " " + p.N + "/" + std::to_string(p.pair ? cols / 2u : cols);
  };
  auto count = [&](uint32_t rows, uint32_t cols) {
    const std::string r = std::to_string(rows) + "u", c = std::to_string(p.pair ? cols / 2u : cols) + "u";
    return "((p.M - 1u) / " + r + " + 1u) * ((p.N - 1u) / " + c + " + 1u)";
  };
  // k in P parts, at least `least` of it in each, where `terms` make fewer than kCUs workgroups.
  auto split = [&](uint32_t least, const std::string& terms, const char* mode) {
    int n = 0;
    std::istringstream in(terms);
    for (std::string t; in >> t;) ++n;
    return "split " + p.K + " " + std::to_string(least) + " " + std::to_string(kCUs) + " " + mode + " " + std::to_string(n) + " " + terms;
  };
  auto parts = [&](uint32_t least, const std::string& blocks) {
    return "tca::hip::col_split(p.K, " + blocks + ", " + std::to_string(least) + "u, " + std::to_string(kCUs) + "u)";
  };
  auto join = [&](const std::string& suffix, uint32_t slices, const std::string& P, const std::string& record,
                  std::vector<std::string> records, const std::string& of) {
    Writer::Kernel j;
    j.suffix = p.suffix + suffix;
    j.params = p.params + " " + part;
    j.block = 32u * slices;
    j.body = ops.str() + "  tca::hip::join_parts<" + pair + ", " + std::to_string(slices) + "u>(" + part + ", epi, p.M, p.N, " + P + ");\n";
    j.grid = p.M + "/1 " + p.N + "/256";
    j.records = std::move(records);
    j.records.push_back(record);
    j.detail = p.what + ", the partial sums of " + of + " (P > 1 only)";
    w->Add(j);
  };
  // The partial sums of kCUs workgroups, of 128x128 results each at most (of few
  // rows 64x64, of a pair twice that): products of one program run in turn and share it.
  if (!w->Has(part)) {
    w->Dim("part_dim", uint64_t{kCUs} * 128u * 128u);
    w->Tensor(part, "f32", "local", "part_dim");
  }

  // A forward product of few rows, at any alignment.
  const bool few = !p.a_rc && p.b_rc;
  if (few) {
    const uint32_t least = 256;  // a step for each wave
    const std::string strips = "((p.N - 1u) / tca::hip::kFewColumns + 1u)", P = parts(least, strips), terms = p.N + "/64";
    uint32_t from = 1;
    for (uint32_t blocks : {1u, 2u, 4u}) {
      Writer::Kernel k;
      k.suffix = p.suffix + "_few" + std::to_string(16u * blocks);
      k.params = p.params + " " + part;
      k.block = 512;
      k.body = ops.str() + "  tca::hip::product_few<" + f16 + ", " + pair + ", " + std::to_string(blocks) + ">(p, epi, " + part + ", " +
               strips + ", " + P + ");\n";
      k.grid = terms;
      k.records = {split(least, terms, "0"), sums, When("M", from, 16u * blocks)};
      k.detail = p.what + ", " + std::to_string(from) + " to " + std::to_string(16u * blocks) + " rows, strips of 64 columns, k over 8 waves and P workgroups";
      w->Add(k);
      from = 16u * blocks + 1u;
    }
    join("_fewjoin", 8, P, split(least, terms, "1"), {When("M", 1, kFewRows)}, "few rows");
  }
  // Rows of whole 16-byte chunks, of both operands, go straight into LDS.
  std::vector<std::string> aligned, odd;
  for (const std::string& d : std::set<std::string>{p.a_rc ? p.M : p.K, p.b_rc ? p.N : p.K}) {
    aligned.push_back(When(d, 0, kMost, 8));
    odd.push_back("unless " + d + " 0 " + std::to_string(kMost) + " 8 0");
  }
  if (few) aligned.push_back(When("M", kFewRows + 1u, kMost));
  if (few) odd.push_back(When("M", kFewRows + 1u, kMost));
  const std::string small_plane = When(plane, 0, kSplitPlane), large_plane = When(plane, kSplitPlane + 1u, 18446744073709551615ull);
  auto with = [](std::vector<std::string> v, std::initializer_list<std::string> r) {
    v.insert(v.end(), r);
    return v;
  };
  const std::string whole = "(p, epi, blockIdx.x, 0u, (p.K + 63u) / 64u * " + std::to_string(p.segs) + "u);\n";
  auto body = [&](const std::string& call) { return ops.str() + "  tca::hip::" + call + whole; };
  // One product of few tiles: `call` on the tile and chunk of k of a workgroup.
  auto few_tiles = [&](const std::string& suffix, const std::string& call, uint32_t block, uint32_t rows, const std::vector<std::string>& records,
                       const std::string& detail) {
    const uint32_t least = 512;  // eight turns
    const std::string P = parts(least, count(rows, 128)), terms = tiles(rows, 128);
    Writer::Kernel k;
    k.suffix = p.suffix + suffix;
    k.params = p.params + " " + part;
    k.block = block;
    k.body = ops.str() + "  const uint32_t tiles = " + count(rows, 128) + ", P = " + P + ";\n" +
             "  const uint32_t chunk = blockIdx.x / tiles;\n  const tca::hip::Run run = tca::hip::run_of(p.K, " +
             std::to_string(p.segs) + "u, chunk, P);\n  tca::hip::" + call + "(p, tca::hip::split_store<" + pair + ">(epi, " + part +
             ", chunk, P, p.M, p.N), blockIdx.x % tiles, run.first, run.end);\n";
    k.grid = terms;
    k.records = with(records, {split(least, terms, "0"), sums, small_plane});
    k.detail = p.what + ", " + detail + ", k over P workgroups (at most " + std::to_string(kSplitPlane) + " results)";
    w->Add(k);
    join(suffix + "join", 4, P, split(least, terms, "1"), with(records, {small_plane}), detail);
  };
  few_tiles("_k", "product_ring<" + targs + ", 128, 64, 2, 2, 5, 5>", 256, 128, aligned, "tiles of 128x128, direct to LDS");
  Writer::Kernel k;
  const std::string cfg_r = "product_ring<" + targs + ", 128, 64, 2, 2, 5, 5>";
  k.suffix = p.suffix + (p.pair ? "_r" : "_t");
  k.params = p.params;
  k.records = with(aligned, {large_plane});
  k.body = body(p.pair ? cfg_r : "product_ring<" + targs + ", 64, 64, 2, 2, 5, 5>");
  k.grid = p.pair ? tiles(128, 128) : tiles(64, 128);
  k.detail = p.what + (p.pair ? ", tiles of 128x128" : ", tiles of 64x128") + " (up to 256x256 where they fill the card), 4 waves, direct to LDS";
  // Larger tiles load less for a product, and need more of the plane to fill
  // 256 CUs; one workgroup of 256x256 or 256x128 holds a CU, two of 128x128 with
  // shorter rings do. Bounds by whole rounds of the card, at k = 4096 (us, bf16, _l /
  // _m / _s / _r; products of k-contiguous and row-contiguous operands and pairs
  // alike within 5%):
  //   tiles of 256x256    64: 79.5 / 50.4 / 39.9 / 36.0   130: 87.3 / 102.6 / 89.5 / 97.0
  //                       96: 82.5 / 53.2 / 53.5 / 64.5   256: 104 / 118 / 121 / 145
  //                      272: 172 / 155 / 167 / 188       384: 191 / 179 / 202 / 244
  //                      400: 187 / 217 / 236 / 274       512: 203 / 242 / 263 / 310
  // Up to 128 tiles of 128x128, tiles of 64x128 put a workgroup on twice as many
  // CUs (_r / 64x128: 2048 x 1024 30.7 / 25.3; 1536 x 1664, 156 tiles, 31.0 / 45.5).
  auto form = [&](Writer::Kernel* of, const char* suffix, const std::string& what, const std::string& call, uint32_t rows,
                  uint32_t cols, uint32_t least, const std::string& terms) {
    // its grid, then the bound: at least so many tiles, of `terms`
    of->forms.push_back({p.suffix + suffix, body(call), p.what + ", " + what,
                         "0 2 1 2 " + tiles(rows, cols) + " " + std::to_string(least) + " 2 " + terms});
  };
  const std::string large = tiles(256, 256), tall = tiles(256, 128), small = tiles(128, 128);
  const std::string what_l = "tiles of 256x256", what_m = "tiles of 256x128", what_s = "tiles of 128x128, two workgroups a CU";
  const std::string ring = "product_ring<" + targs;
  const std::string cfg_l = ring + ", 256, 128, 2, 2, 3, 2>", cfg_m = ring + ", 256, 64, 2, 2, 3, 3>", cfg_s = ring + ", 128, 64, 2, 2, 3, 2>";
  form(&k, "_l", what_l, cfg_l, 256, 256, 385, large);
  form(&k, "_m", what_m, cfg_m, 256, 128, 257, large);
  form(&k, "_l", what_l, cfg_l, 256, 256, 257, tall);
  form(&k, "_m", what_m, cfg_m, 256, 128, 192, tall);
  form(&k, "_s", what_s, cfg_s, 128, 128, 257, small);
  if (!p.pair) form(&k, "_r", "tiles of 128x128, one workgroup a CU", cfg_r, 128, 128, 129, small);
  w->Add(k);
  // (1101 x 1001 x 2049, 72 tiles of 128x128: 34 us, of 64x128 27; 132 of them 35 and
  // 36; 432, 53 and 70.)
  few_tiles("_o", "product_any<" + targs + ", 64>", 512, 64, odd, "tiles of 64x128, any shape and alignment");
  const std::string what_a = "tiles of 128x128, any shape and alignment", cfg_a = "product_any<" + targs + ", 128>";
  Writer::Kernel any;
  any.params = p.params;
  any.block = 512;
  // Two workgroups a CU (bf16 4001 x 2049 x 3203 111 us with one, 97 so; 1501 x 1003 x
  // 1701, 168 tiles, 19 either way; what spills is read again outside
  // the loop, but for rows of less than 8).
  any.waves = 4;
  any.records = with(odd, {large_plane});
  if (p.pair) {  // 128 tiles and more
    any.suffix = p.suffix + "_a";
    any.body = body(cfg_a);
    any.grid = small;
    any.detail = p.what + ", " + what_a;
  } else {
    any.suffix = p.suffix;
    any.body = body("product_any<" + targs + ", 64>");
    any.grid = tiles(64, 128);
    any.detail = p.what + ", tiles of 64x128 (128x128 from 128 tiles on), any shape and alignment";
    form(&any, "_a", what_a, cfg_a, 128, 128, 128, small);
  }
  w->Add(any);
}

void EmitForward(const Attrs& a, bool gated, Writer* w) {
  const bool bias = a.Flag("bias"), res = a.Flag("residual"), save = a.Flag("save");
  const std::string T = ElemType(a.elem), act = std::to_string(ActCode(a.act)), none = "(" + T + "*)nullptr";
  w->Header("tca/hip/product.h");
  for (const char* d : {"M", "K", "N"}) w->Dim(d);
  w->Tensor("x", a.elem, "in", "M K");
  Product p;
  p.M = "M";
  p.N = "N";
  p.K = "K";
  p.A[0] = "x";
  p.b_rc = true;
  std::string params;
  if (gated) {
    w->Tensor("wg", a.elem, "in", "K N");
    w->Tensor("wu", a.elem, "in", "K N");
    if (bias) w->Tensor("bg", a.elem, "in", "N");
    if (bias) w->Tensor("bu", a.elem, "in", "N");
    w->Tensor("h", a.elem, "out", "M N");
    if (save) w->Tensor("g", a.elem, "out", "M N");
    if (save) w->Tensor("u", a.elem, "out", "M N");
    p.pair = true;
    p.B[0][0] = "wg";
    p.B[1][0] = "wu";
    p.params = std::string("x wg wu ") + (bias ? "bg bu " : "") + "h " + (save ? "g u " : "") + "M K N";
    p.epi = "tca::hip::GatedStore<" + T + ", " + act + ", " + Bool(bias) + ", " + Bool(save) + ">{" +
            (bias ? "bg, bu" : none + ", " + none) + ", h, " + (save ? "g, u" : none + ", " + none) + ", N}";
    p.what = "gated projections, " + a.act;
  } else {
    w->Tensor("w", a.elem, "in", "K N");
    if (bias) w->Tensor("b", a.elem, "in", "N");
    if (res) w->Tensor("res", a.elem, "in", "M N");
    w->Tensor("y", a.elem, "out", "M N");
    if (save) w->Tensor("z", a.elem, "out", "M N");
    p.B[0][0] = "w";
    p.params = std::string("x w ") + (bias ? "b " : "") + (res ? "res " : "") + "y " + (save ? "z " : "") + "M K N";
    p.epi = "tca::hip::LinearStore<" + T + ", " + act + ", " + Bool(bias) + ", " + Bool(res) + ", " + Bool(save) + ">{" +
            (bias ? "b" : none) + ", " + (res ? "res" : none) + ", y, " + (save ? "z" : none) + ", N}";
    p.what = "projection, " + a.act;
  }
  EmitProduct(a, p, w);
}

void EmitBackward(const Attrs& a, bool gated, Writer* w) {
  const bool bias = a.Flag("bias"), slope = gated || a.act != "none";
  const std::string T = ElemType(a.elem), act = std::to_string(ActCode(a.act)), none = "(" + T + "*)nullptr";
  w->Header("tca/hip/product.h");
  for (const char* d : {"M", "K", "N"}) w->Dim(d);
  // Partial rows of the bias' gradient: one for each kPartRows rows of the batch, at most kParts.
  const uint32_t kParts = 256, kPartRows = 16;
  if (bias) w->Dim("parts", kParts);
  if (bias) w->Dim("grads", gated ? 2 : 1);
  w->Tensor(gated ? "dh" : "dy", a.elem, "in", "M N");
  w->Tensor("x", a.elem, "in", "M K");
  for (const char* t : {"wg", "wu"})
    if (gated) w->Tensor(t, a.elem, "in", "K N");
  if (!gated) w->Tensor("w", a.elem, "in", "K N");
  for (const char* t : {"g", "u"})
    if (gated) w->Tensor(t, a.elem, "in", "M N");
  if (!gated && slope) w->Tensor("z", a.elem, "in", "M N");
  for (const char* t : {"dg", "du"})
    if (gated) w->Tensor(t, a.elem, "out", "M N");
  if (!gated && slope) w->Tensor("dz", a.elem, "out", "M N");
  w->Tensor("dx", a.elem, "out", "M K");
  for (const char* t : {"dwg", "dwu"})
    if (gated) w->Tensor(t, a.elem, "out", "K N");
  if (!gated) w->Tensor("dw", a.elem, "out", "K N");
  for (const char* t : {"dbg", "dbu"})
    if (gated && bias) w->Tensor(t, a.elem, "out", "N");
  if (!gated && bias) w->Tensor("db", a.elem, "out", "N");
  if (bias) w->Tensor("bias_part", "f32", "local", "parts grads N");

  // The gradients of the pre-activations.
  const std::string f = "  const tca::hip::Slope<" + T + ", " + act + ", " + Bool(gated) + "> f{" +
                        (gated ? "dh, g, u, dg, du" : slope ? "dy, z, " + none + ", dz, " + none
                                                            : "dy, " + none + ", " + none + ", " + none + ", " + none) + "};\n";
  const std::string tensors = gated ? "dh g u dg du " : slope ? "dy z dz " : "dy ";
  const std::string parts = "tca::hip::partial_rows(M, " + std::to_string(kPartRows) + "u, " + std::to_string(kParts) + "u)";
  if (bias) {
    Writer::Kernel k;
    k.suffix = "_slope";
    k.params = tensors + "bias_part M N";
    k.block = 1024;
    k.body = f + "  tca::hip::slope_columns(f, bias_part, M, N, " + parts + ");\n";
    k.grid = "N/512 M/" + std::to_string(kPartRows) + ":" + std::to_string(kParts);
    k.records = {Scratch("bias_part", "M/" + std::to_string(kPartRows) + ":" + std::to_string(kParts) + " N/1" +
                                          (gated ? " 2/1" : ""))};
    k.detail = "gradients of the pre-activations, partial sums of the bias' gradient";
    w->Add(k);
    Writer::Kernel j;
    j.suffix = "_bias";
    j.params = std::string("bias_part ") + (gated ? "dbg dbu " : "db ") + "M N";
    j.body = "  tca::hip::join_partials<" + T + ">(bias_part, " + (gated ? "dbg, dbu, 2u" : "db, " + none + ", 1u") + ", N, " + parts + ");\n";
    j.block = 1024;
    j.grid = std::string("N/32") + (gated ? " 2/1" : "");
    j.detail = "the bias' gradient from its partial sums";
    w->Add(j);
  } else if (slope) {
    Writer::Kernel k;
    k.suffix = "_slope";
    k.params = tensors + "M N";
    k.body = f + "  tca::hip::slope_flat(f, M * N);\n";
    k.grid = "M*N/2048";
    k.detail = "gradients of the pre-activations";
    w->Add(k);
  }
  const std::string dz = gated ? "dg" : slope ? "dz" : "dy";
  // dx = dz w^T: the rows of the weight are the columns of its product.
  Product x;
  x.suffix = "_dx";
  x.what = "the input's gradient";
  x.M = "M";
  x.N = "K";
  x.K = "N";
  x.A[0] = dz;
  x.A[1] = "du";
  x.B[0][0] = gated ? "wg" : "w";
  x.B[0][1] = "wu";
  x.segs = gated ? 2 : 1;
  x.params = dz + (gated ? " du wg wu" : " w") + " dx M K N";
  x.epi = "tca::hip::PlainStore<" + T + ">{dx, " + none + ", K}";
  EmitProduct(a, x, w);
  // dw = x^T dz: both run over their rows.
  Product d;
  d.suffix = "_dw";
  d.what = "the weights' gradient";
  d.M = "K";
  d.N = "N";
  d.K = "M";
  d.A[0] = "x";
  d.B[0][0] = dz;
  d.B[1][0] = "du";
  d.a_rc = d.b_rc = true;
  d.pair = gated;
  d.params = "x " + dz + (gated ? " du dwg dwu" : " dw") + " M K N";
  d.epi = "tca::hip::PlainStore<" + T + ">{" + (gated ? "dwg, dwu" : "dw, " + none) + ", N}";
  EmitProduct(a, d, w);
}

// ------------------------------------------- positions and paged attention

void EmitPageTable(Writer* w) {
  w->Header("tca/hip/positions.h");
  for (const char* d : {"S", "S1", "F", "one", "P", "T"}) w->Dim(d, std::string(d) == "one" ? 1 : 0);
  w->Dim("page");
  w->List("held", "i32", "in", "S");
  w->List("fresh", "i32", "in", "S");
  w->List("free_pages", "i32", "in", "F");
  w->List("first", "i32", "in", "one");
  w->List("table", "i32", "out", "S P");
  w->List("starts", "i32", "out", "S1");
  w->List("lens", "i32", "out", "S");
  w->List("pos", "i32", "out", "T");
  w->List("slot", "i32", "out", "T");
  w->List("next", "i32", "out", "one");
  w->Require("eq 1 S1/1 2 S/1 1/1");
  w->Require("le 1 1/1 1 page/1");
  Writer::Kernel k;
  k.params = "held fresh free_pages first table starts lens pos slot next S F P T page";
  k.block = 1024;
  k.body = "  tca::hip::page_table(held, fresh, free_pages, first, table, starts, lens, pos, slot, next, S, F, P, T, page);\n";
  k.grid = "1/1";
  k.detail = "block tables and slot maps, 1024 runs of sequences added up in every workgroup";
  // Every workgroup adds up all sequences, so at most 256 of them place tokens.
  k.forms.push_back({"_many", k.body, "the same, on several workgroups", "0 1 2 1 T/1024:256"});
  w->Add(k);
}

// Tokens of a workgroup: four where a token has at most kRotaryNarrow values and there
// are kRotaryMany (bf16 [16384, 8, 64]: 9.9 us with one, 6.7 with four; [8192, 32, 128] 21.0
// and 21.6, [2048, 40, 128] 7.3 and 8.0, [64, 40, 128] 3.0 and 4.5).
constexpr uint32_t kRotaryTokens = 4, kRotaryNarrow = 1024, kRotaryMany = 2048;

void EmitRotary(const Attrs& a, bool cache, Writer* w) {
  w->Header("tca/hip/positions.h");
  if (cache) {
    for (const char* d : {"T", "H", "D", "F", "HK", "G", "PAGES", "PAGE"}) w->Dim(d);
    w->Tensor("x", a.elem, "in", "T H D");
    w->List("pos", "i32", "in", "T");
    w->List("slot", "i32", "in", "T");
    w->List("freq", "f32", "in", "F");
    w->Tensor("q", a.elem, "out", "T HK G D");
    w->Tensor("k", a.elem, "out", "PAGES HK PAGE D");
    w->Tensor("v", a.elem, "out", "PAGES HK PAGE D");
    w->Require("eq 1 H/1 2 HK*G/1 2*HK/1");
  } else {
    for (const char* d : {"T", "H", "D", "F"}) w->Dim(d);
    w->Tensor("x", a.elem, "in", "T H D");
    w->List("pos", "i32", "in", "T");
    w->List("freq", "f32", "in", "F");
    w->Tensor("y", a.elem, "out", "T H D");
  }
  w->Require("le 1 2*F/1 1 D/1");
  w->Require("le 1 F/1 1 512/1");
  w->Scalar("scale");
  const std::string T = ElemType(a.elem), inter = Bool(a.Flag("interleaved")), inverse = Bool(a.Flag("inverse"));
  auto body = [&](uint32_t tokens) {
    return cache ? "  tca::hip::rotary_cache<" + T + ", " + inter + ", " + std::to_string(tokens) +
                       ">(x, pos, slot, freq, q, k, v, T, HK, G, D, F, PAGES, PAGE, scale);\n"
                 : "  tca::hip::rotary<" + T + ", " + inter + ", " + inverse + ", " + std::to_string(tokens) +
                       ">(x, pos, freq, y, T, H, D, F, scale);\n";
  };
  const std::string what = cache ? "rotary positions, keys and values stored into the cache's pages" : "rotary positions";
  Writer::Kernel k;
  k.params = cache ? "x pos slot freq q k v T HK G D F PAGES PAGE scale" : "x pos freq y T H D F scale";
  k.body = body(1);
  k.grid = "T/1 H*D/1:1";
  k.records = {When("H*D", kRotaryNarrow + 1u, 18446744073709551615ull)};
  k.detail = what + ", a token a workgroup";
  w->Add(k);
  k.suffix = "_narrow";
  k.records = {When("H*D", 0, kRotaryNarrow)};
  k.detail = what + " of at most " + std::to_string(kRotaryNarrow) + " values a token";
  k.forms.push_back({"_t4", body(kRotaryTokens), k.detail + ", four tokens a workgroup",
                     "0 2 1 2 T/" + std::to_string(kRotaryTokens) + " H*D/1:1 " + std::to_string(kRotaryMany) + " 1 T/1"});
  w->Add(k);
}

void EmitPagedAttention(const Attrs& a, Writer* w) {
  const bool stats = a.Flag("stats"), window = a.Flag("window");
  w->Header("tca/hip/attention.h");
  for (const char* d : {"T", "HK", "G", "D", "PAGES", "PAGE", "S", "P", "S1"}) w->Dim(d);
  if (window) w->Dim("window");
  // Two parts of a tile for each of 256 workgroups.
  w->Dim("slots", 512);
  w->Dim("few_rows", 32);
  w->Dim("many_rows", 256);
  w->Dim("wide_rows", 128);  // of tiles of heads above 128
  w->Dim("pair", 2);
  w->Dim("groups", 256);
  w->Dim("words", 8);
  w->Tensor("q", a.elem, "in", "T HK G D");
  w->Tensor("k", a.elem, "in", "PAGES HK PAGE D");
  w->Tensor("v", a.elem, "in", "PAGES HK PAGE D");
  w->List("table", "i32", "in", "S P");
  w->List("starts", "i32", "in", "S1");
  w->List("lens", "i32", "in", "S");
  w->Tensor("y", a.elem, "out", "T HK G D");
  if (stats) w->List("lse", "f32", "out", "T HK G");
  w->Tensor("few_part", "f32", "local", "slots few_rows D");
  w->Tensor("few_ml", "f32", "local", "slots few_rows pair");
  w->Tensor("many_part", "f32", "local", "slots many_rows D");
  w->Tensor("many_ml", "f32", "local", "slots many_rows pair");
  w->Tensor("wide_part", "f32", "local", "slots wide_rows D");
  w->Tensor("wide_ml", "f32", "local", "slots wide_rows pair");
  w->Tensor("few_join", "u32", "local", "groups words");
  w->Tensor("many_join", "u32", "local", "groups words");
  w->Scalar("scale");
  w->Require("eq 1 S1/1 2 S/1 1/1");
  w->Require("mod 1 D/1 1 8/1");
  w->Require("le 1 8/1 1 D/1");
  w->Require("le 1 D/1 1 256/1");
  if (window) w->Require("le 1 1/1 1 window/1");
  const std::string T = ElemType(a.elem), f16 = Bool(a.elem == "f16");
  uint32_t from = 0;
  for (uint32_t dp : {64u, 128u, 192u, 256u}) {
    const std::string DP = std::to_string(dp);
    const uint32_t rows = dp <= 128u ? 256u : 128u;
    const std::string big = dp <= 128u ? "many" : "wide";  // whose locals: a launch allocates those that its kernels take
    const std::string head = "  const tca::hip::AttendShape a = {table, starts, lens, T, HK, G, D, PAGES, PAGE, S, P, " +
                             std::string(window ? "window" : "0u") + "};\n";
    auto out = [&](const std::string& name, const std::string& parts, uint32_t most) {
      return std::string("  const tca::hip::AttendOut<") + T + "> " + name + " = {y, " + (stats ? "lse" : "(float*)nullptr") + ", " + parts +
             "_part, reinterpret_cast<float2*>(" + parts + "_ml), " + name + "_join, tca::hip::attend_part_rows(T, G, " + std::to_string(most) +
             "u)};\n";
    };
    const std::string outs = out("few", "few", 32) + out("many", big, rows);
    auto records = [&]() {
      std::vector<std::string> r = {When("D", from, dp)};
      for (const std::string& n : {std::string("few"), big}) {
        const std::string most = std::to_string(n == "few" ? 32u : rows);
        r.push_back(Scratch(n + "_part", "512/1 T*G/1:" + most + " D/1"));
        r.push_back(Scratch(n + "_ml", "1024/1 T*G/1:" + most));
      }
      return r;
    };
    const std::string written = std::string("y ") + (stats ? "lse " : "") + "few_part few_ml " + big + "_part " + big + "_ml few_join many_join T HK G D";
    Writer::Kernel k;
    k.suffix = "_" + DP;
    k.params = "q k v table starts lens " + written + " PAGES PAGE S P" + (window ? " window" : "") + " scale";
    k.body = head + outs + "  tca::hip::attend<" + f16 + ", " + DP +
             ">(a, q, k, v, reinterpret_cast<const uint4*>(tca::hip::kAttendZero), few, many, scale);\n";
    k.grid = "256/1 T*HK/1:1 G/1:1";
    k.block = dp <= 128u ? 512 : 256;
    k.waves = dp <= 128u ? 2 : 1;
    k.records = records();
    k.detail = "attention over pages, heads of " + std::to_string(from) + " to " + DP + ", equal runs of key blocks on 256 workgroups";
    w->Add(k);
    Writer::Kernel j;
    j.suffix = "_" + DP + "join";
    j.params = k.params;
    j.waves = 6;  // the join's loads in flight: what follows a flagged tile would take more registers
    j.body = head + outs + "  tca::hip::join_attention<" + f16 + ", " + DP + ">(a, q, k, v, few, many, scale);\n";
    // Workgroups of a tile: one for each 256 of its four-column pieces, at most 8 (prompts of
    // 4096: 57 us with one, 17 with 8).
    j.grid = "256/1 T*G*D/1024:8 HK/1:1";
    j.records = records();
    j.detail = "the parts of tiles that several workgroups share";
    w->Add(j);
    from = dp + 1u;
  }
}

}  // namespace

OpStatus EmitOperator(const std::string& name, const std::string& attributes, const std::string& target, Result* out,
                      std::string* program, std::string* err) {
  const Spec* spec = nullptr;
  for (const auto& s : Specs())
    if (name == s.name) spec = &s;
  if (spec == nullptr) {
    *err = "no operator " + name + "; there are:\n" + ListOperators();
    return OpStatus::NoSuchOperator;
  }
  if (target != "gfx950") {
    *err = "operator " + name + ": unsupported target " + target + " (gfx950 only)";
    return OpStatus::Unsupported;
  }
  Attrs a;
  if (!ParseAttrs(*spec, attributes, &a, err)) return OpStatus::Unsupported;
  // Attributes in a fixed order: one program, one name, however they are written.
  std::string full = name + (a.elem.empty() ? "" : "_" + a.elem);
  if (spec->weight && a.weight != a.elem) full += "_w" + a.weight;
  if (spec->act) full += "_" + a.act;
  for (const auto& f : Flags(*spec))
    if (a.Flag(f.c_str())) full += "_" + f;
  Writer w(full);
  if (name == "layer_norm") EmitLayerNorm(a, &w);
  else if (name == "layer_norm_backward") EmitLayerNormBackward(a, &w);
  else if (name == "linear") EmitForward(a, false, &w);
  else if (name == "gated") EmitForward(a, true, &w);
  else if (name == "linear_backward") EmitBackward(a, false, &w);
  else if (name == "gated_backward") EmitBackward(a, true, &w);
  else if (name == "page_table") EmitPageTable(&w);
  else if (name == "paged_attention") EmitPagedAttention(a, &w);
  else EmitRotary(a, name == "rotary_cache", &w);
  w.Finish(target, out);
  *program = full;
  return OpStatus::Ok;
}

std::string ListOperators() {
  std::string s;
  for (const auto& x : Specs()) s += std::string(x.name) + " " + Usage(x) + "\n";
  return s;
}

}  // namespace cg
}  // namespace tca
