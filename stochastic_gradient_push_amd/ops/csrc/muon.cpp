// Newton-Schulz and Muon entry points: argument checks, outputs and
// workspace for muon_kernels.hip.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include "call_checks.h"

extern "C" {
int sgp_ns_chunk();
int64_t sgp_ns_plan_big_tiles(int64_t tiles, bool sym);
bool sgp_ns_is_small(int n, int m);
void sgp_newton_schulz(int dtype, const void* g, void* out, const void* mat,
                       int batch, int steps, int split_steps, int group,
                       float a, float b, float c, float growth, float eps,
                       void* work, double* partials, float* r,
                       hipStream_t s);
void sgp_muon_step(int dtype, float* p, const void* g, float* buf,
                   void* shadow, const float* lr, float mu, float wd,
                   float rest_lr, bool nesterov, int steps, int group, float a,
                   float b, float c, float growth, float eps, const void* tables,
                   const int64_t* layout, void* work, double* partials,
                   float* r, hipStream_t s);
}

namespace {

// the kernels' records, as muon_kernels.hip has them
struct Mat {
  int64_t start, x_off, a_off;
  int rows, cols, n, m, np, mp, chunk0, chunk1;
  int e;
  float scale;
};
struct Tile { int mat, tm, tn, big; };
struct Task {
  Mat q;
  Tile t;
};
struct Chunk { int64_t start; int count, mat; };

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A side is at most 2^15 (n m entries of 1 / sqrt(n m) times 2^e around 1,
// e up to 13) and a matrix at most 2^30 values.
void check_matrix(int64_t rows, int64_t cols) {
  TORCH_CHECK(rows >= 1 && cols >= 1 && rows <= (1 << 20)
              && cols <= (1 << 20) && rows * cols <= (int64_t(1) << 30)
              && std::min(rows, cols) <= (1 << 15),
              "newton_schulz: a matrix must have 1 to 2^20 rows and columns, "
              "one of them at most 2^15, and at most 2^30 values, got ",
              rows, " x ", cols);
}

Mat make_mat(int64_t start, int64_t rows, int64_t cols, double scale) {
  Mat q{};
  q.start = start;
  q.rows = (int)rows;
  q.cols = (int)cols;
  q.n = (int)std::min(rows, cols);
  q.m = (int)std::max(rows, cols);
  q.np = (int)(cdiv(q.n, 64) * 64);
  q.mp = (int)(cdiv(q.m, 64) * 64);
  q.chunk1 = (int)cdiv(rows * cols, sgp_ns_chunk());
  q.e = std::min(13, std::ilogb(std::sqrt((double)rows * (double)cols)));
  q.scale = (float)scale;
  return q;
}

// fp16 values of workspace: X and its transpose twice and five matrices of
// A's size, two planes each
int64_t work_size(int64_t x_total, int64_t a_total) {
  return 8 * x_total + 10 * a_total;
}

int dtype_code(const torch::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return 0;
    case torch::kBFloat16: return 1;
    case torch::kFloat16: return 2;
    default:
      TORCH_CHECK(false, what, " must be fp32, bf16 or fp16, got ",
                  t.scalar_type());
  }
}

hipStream_t stream_of(const torch::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// g: [batch, rows, cols]
torch::Tensor newton_schulz(const torch::Tensor& g, int64_t steps,
                            int64_t split_steps, int64_t group, double a,
                            double b, double c, double growth, double eps) {
  check_untraced("newton_schulz");
  check_tangent("newton_schulz", g);
  TORCH_CHECK(g.is_cuda() && g.is_contiguous() && g.dim() == 3,
              "newton_schulz: g must be a contiguous [batch, rows, cols] "
              "device tensor");
  const int dtype = dtype_code(g, "newton_schulz: g");
  check_memory("newton_schulz", g);
  TORCH_CHECK(steps >= 1 && steps <= 100 && split_steps >= 0
              && split_steps <= steps && group >= 1,
              "newton_schulz: steps out of range");
  const c10::DeviceGuard guard(g.device());
  torch::Tensor out = torch::empty_like(g);
  check_memory("newton_schulz", out);  // under a mode that makes such tensors
  if (g.numel() == 0) return out;
  const int64_t batch = g.size(0);
  check_matrix(g.size(1), g.size(2));
  const Mat q = make_mat(0, g.size(1), g.size(2), 1.0);
  const int64_t x_total = batch * q.np * (int64_t)q.mp;
  const int64_t a_total = batch * q.np * (int64_t)q.np;
  const bool small = sgp_ns_is_small(q.n, q.m);
  // matrices and chunks are counted in 32 bits, and a launch has less than
  // 2^32 threads, 256 a tile or chunk (such a workspace would fill the card
  // several times); small matrices are launched in parts
  TORCH_CHECK(batch * q.chunk1 < (int64_t(1) << 31)
              && (small || (x_total / 4096 < (int64_t(1) << 24)
                            && batch * q.chunk1 < (int64_t(1) << 24))),
              "newton_schulz: too many values in one call");
  torch::Tensor work, partials, r;
  if (!small) {
    const auto opt = g.options();
    work = torch::empty({work_size(x_total, a_total)},
                        opt.dtype(torch::kFloat16));
    partials = torch::empty({batch * q.chunk1}, opt.dtype(torch::kFloat64));
    r = torch::empty({batch}, opt.dtype(torch::kFloat32));
  }
  sgp_newton_schulz(dtype, g.data_ptr(), out.data_ptr(), &q, (int)batch,
                    (int)steps, (int)split_steps, (int)group, (float)a,
                    (float)b, (float)c, (float)growth, (float)eps,
                    work.defined() ? work.data_ptr() : nullptr,
                    work.defined() ? partials.data_ptr<double>() : nullptr,
                    work.defined() ? r.data_ptr<float>() : nullptr,
                    stream_of(g));
  C10_HIP_CHECK(hipGetLastError());
  return out;
}

// The tiles of one product of all matrices: X X^T or A^2 (sym: on and above
// the diagonal) or B X.  As many 128 x 128 tiles as fill the card, the
// longest sums first, so that what starts last ends soon; of sums of one
// length the tiles that one XCD gets (every eighth block) are neighbours: in
// one matrix, or in few.
std::vector<Tile> product_tiles(const std::vector<Mat>& m, bool sym) {
  auto length = [&](const Tile& t) { return sym ? m[t.mat].mp : m[t.mat].np; };
  auto longer = [&](const Tile& x, const Tile& y) {
    return length(x) > length(y);
  };
  std::vector<Tile> big, small;
  for (int i = 0; i < (int)m.size(); ++i) {
    const int nt = m[i].np / 64, mt = sym ? nt : m[i].mp / 64;
    // four pairs of rows at a time, down before to the right
    for (int top = 0; top < nt; top += 8)
      for (int tn = 0; tn < mt; tn += 2)
        for (int tm = top; tm < std::min(top + 8, nt); tm += 2) {
          if (sym && tm > tn) continue;
          if (tm + 1 < nt && tn + 1 < mt) {
            big.push_back({i, tm, tn, 1});
            continue;
          }
          for (int k = 0; k < 4; ++k) {
            const Tile t{i, tm + (k & 1), tn + (k >> 1), 0};
            if (t.tm < nt && t.tn < mt && !(sym && t.tm > t.tn))
              small.push_back(t);
          }
        }
  }
  std::stable_sort(big.begin(), big.end(), longer);
  const size_t keep =
      (size_t)sgp_ns_plan_big_tiles((int64_t)big.size(), sym);
  for (size_t i = keep; i < big.size(); ++i)
    for (int k = 0; k < 4; ++k) {
      const Tile t{big[i].mat, big[i].tm + (k & 1), big[i].tn + (k >> 1), 0};
      if (!(sym && t.tm > t.tn)) small.push_back(t);
    }
  big.resize(keep);
  std::stable_sort(small.begin(), small.end(), [&](const Tile& x,
                                                   const Tile& y) {
    return length(x) != length(y) ? length(x) > length(y) : x.mat < y.mat;
  });
  big.insert(big.end(), small.begin(), small.end());
  for (size_t from = 0; from < big.size();) {
    size_t to = from;
    while (to < big.size() && length(big[to]) == length(big[from])
           && big[to].big == big[from].big)
      ++to;
    const std::vector<Tile> part(big.begin() + from, big.begin() + to);
    size_t k = 0;
    for (size_t xcd = 0; xcd < 8; ++xcd)
      for (size_t at = from + (xcd + 8 - from % 8) % 8; at < to; at += 8)
        big[at] = part[k++];
    from = to;
  }
  return big;
}

// The tables of a Muon step over a flat buffer of `total` values with
// matrices (start, rows, cols, scale); everything between is the rest.
// -> (uint8 tensor on the host, layout)
std::tuple<torch::Tensor, std::vector<int64_t>> muon_plan(
    const std::vector<std::tuple<int64_t, int64_t, int64_t, double>>& mats,
    int64_t total) {
  for (const auto& [start, rows, cols, scale] : mats)
    check_matrix(rows, cols);
  const int chunk = sgp_ns_chunk();
  std::vector<Mat> m;
  std::vector<Chunk> chunks;
  std::vector<Tile> pack_tiles;
  std::vector<std::pair<int64_t, int64_t>> taken;
  int64_t x_total = 0, a_total = 0, sum_nnm = 0, sum_nnn = 0;
  for (const auto& [start, rows, cols, scale] : mats) {
    TORCH_CHECK(start >= 0 && start + rows * cols <= total,
                "muon: a matrix lies outside the flat buffer");
    Mat q = make_mat(start, rows, cols, scale);
    q.x_off = x_total;
    q.a_off = a_total;
    q.chunk0 = (int)chunks.size();
    q.chunk1 += q.chunk0;
    const int i = (int)m.size();
    for (int64_t at = 0; at < rows * cols; at += chunk)
      chunks.push_back({start + at,
                        (int)std::min<int64_t>(chunk, rows * cols - at), i});
    x_total += q.np * (int64_t)q.mp;
    a_total += q.np * (int64_t)q.np;
    sum_nnm += (int64_t)q.np * q.np * q.mp;
    sum_nnn += (int64_t)q.np * q.np * q.np;
    for (int tm = 0; tm < q.np / 64; ++tm)
      for (int tn = 0; tn < q.mp / 64; ++tn)
        pack_tiles.push_back({i, tm, tn, 0});
    taken.push_back({start, start + rows * cols});
    m.push_back(q);
  }
  auto tasks = [&](const std::vector<Tile>& tiles) {
    std::vector<Task> v;
    for (const Tile& t : tiles) v.push_back({m[t.mat], t});
    return v;
  };
  const std::vector<Task> packs = tasks(pack_tiles),
                          syms = tasks(product_tiles(m, true)),
                          rects = tasks(product_tiles(m, false));
  std::sort(taken.begin(), taken.end());
  int64_t at = 0;
  auto rest = [&](int64_t to) {
    for (; at < to; at += chunk)
      chunks.push_back({at, (int)std::min<int64_t>(chunk, to - at), -1});
  };
  for (const auto& [from, to] : taken) {
    TORCH_CHECK(from >= at, "muon: two matrices overlap");
    rest(from);
    at = to;
  }
  rest(total);
  // a launch has less than 2^32 threads, 256 a tile or chunk
  TORCH_CHECK(packs.size() < (size_t(1) << 24)
              && chunks.size() < (size_t(1) << 24),
              "muon: too many values in one plan");

  const std::vector<int64_t> layout = {
      (int64_t)m.size(), (int64_t)chunks.size(), (int64_t)packs.size(),
      (int64_t)syms.size(), (int64_t)rects.size(), x_total, a_total,
      sum_nnm, sum_nnn};
  auto bytes = [](const auto& v) { return v.size() * sizeof(v[0]); };
  torch::Tensor tables = torch::empty(
      {(int64_t)(bytes(chunks) + bytes(packs) + bytes(syms)
                 + bytes(rects))},
      torch::TensorOptions().dtype(torch::kUInt8));
  uint8_t* to = tables.data_ptr<uint8_t>();
  auto copy = [&](const auto& v) {
    if (!v.empty()) std::memcpy(to, v.data(), bytes(v));
    to += bytes(v);
  };
  copy(chunks);
  copy(packs);
  copy(syms);
  copy(rects);
  return {tables, layout};
}

void check_flat(const torch::Tensor& t, const char* name,
                const torch::Tensor& p, torch::ScalarType dtype) {
  TORCH_CHECK(t.is_cuda() && t.device() == p.device() && t.is_contiguous()
              && t.dim() == 1 && t.numel() == p.numel()
              && t.scalar_type() == dtype, "muon_step_: ", name,
              " must be a contiguous ", dtype, " vector of ", p.numel(),
              " values on the parameters' device");
  check_memory("muon_step_", t);
}

void muon_step_(torch::Tensor p, const torch::Tensor& g, torch::Tensor buf,
                torch::optional<torch::Tensor> shadow,
                const torch::Tensor& tables,
                const std::vector<int64_t>& layout, int64_t total,
                const torch::Tensor& lr, double momentum, double weight_decay,
                double rest_lr, bool nesterov, int64_t steps, int64_t group,
                double a, double b, double c, double growth, double eps) {
  check_untraced("muon_step_");
  for (const torch::Tensor& t : {p, g, buf, lr})
    check_tangent("muon_step_", t);
  if (shadow.has_value()) check_tangent("muon_step_", *shadow);
  check_flat(p, "params", p, torch::kFloat32);
  TORCH_CHECK(p.numel() == total, "muon_step_: the plan is for ", total,
              " values, params has ", p.numel());
  TORCH_CHECK(g.scalar_type() == torch::kFloat32
              || g.scalar_type() == torch::kBFloat16,
              "muon_step_: grads must be fp32 or bf16, got ",
              g.scalar_type());
  check_flat(g, "grads", p, g.scalar_type());
  check_flat(buf, "momentum_buf", p, torch::kFloat32);
  if (shadow.has_value())
    check_flat(*shadow, "shadow", p, torch::kBFloat16);
  TORCH_CHECK(lr.is_cuda() && lr.device() == p.device() && lr.numel() == 1
              && lr.scalar_type() == torch::kFloat32,
              "muon_step_: lr must be one fp32 value on the parameters' "
              "device");
  check_memory("muon_step_", lr);
  check_memory("muon_step_", tables);
  TORCH_CHECK(tables.device() == p.device(),
              "muon_step_: the plan is for another device");
  TORCH_CHECK(layout.size() == 9, "muon_step_: not a plan");
  TORCH_CHECK(steps >= 1 && steps <= 100 && group >= 1,
              "muon_step_: steps out of range");
  const c10::DeviceGuard guard(p.device());
  const auto opt = p.options();
  torch::Tensor work = torch::empty({work_size(layout[5], layout[6])},
                                    opt.dtype(torch::kFloat16));
  torch::Tensor partials = torch::empty({std::max<int64_t>(1, layout[1])},
                                        opt.dtype(torch::kFloat64));
  torch::Tensor r = torch::empty({std::max<int64_t>(1, layout[0])}, opt);
  // under a mode that makes such tensors
  for (const torch::Tensor& t : {work, partials, r})
    check_memory("muon_step_", t);
  sgp_muon_step(g.scalar_type() == torch::kFloat32 ? 0 : 1,
                p.data_ptr<float>(), g.data_ptr(), buf.data_ptr<float>(),
                shadow.has_value() ? shadow->data_ptr() : nullptr,
                lr.data_ptr<float>(), (float)momentum, (float)weight_decay,
                (float)rest_lr, nesterov, (int)steps, (int)group, (float)a,
                (float)b, (float)c, (float)growth, (float)eps, tables.data_ptr(),
                layout.data(), work.data_ptr(), partials.data_ptr<double>(),
                r.data_ptr<float>(), stream_of(p));
  C10_HIP_CHECK(hipGetLastError());
}

}  // namespace

void init_muon(py::module_& m) {
  m.def("newton_schulz", &newton_schulz,
        "orthogonal factors of [batch, rows, cols] by Newton-Schulz steps");
  m.def("muon_plan", &muon_plan,
        "tables of a Muon step: (start, rows, cols, scale) of each matrix");
  m.def("muon_step_", &muon_step_,
        "momentum, Newton-Schulz and update over a flat buffer");
}
