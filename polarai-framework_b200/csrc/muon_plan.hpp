// The order of orthogonalised momentum's products: which operations a matrix's rounds are made of, and which of them share a launch.  Host
// code without CUDA, so that it is tested without a GPU.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <utility>
#include <vector>

namespace polar_b200 {
namespace muon {

constexpr float kX = 32768.f, kG = 32768.f, kP = 16384.f;  // what X, G and P are held times
constexpr float kQ = 4096.f;                               // and the product of two P: kBoundP^2 * 2^12 is below 65504
constexpr uint64_t kNarrow = 128;                          // a short side up to here fits the kernel that does all symmetric products of a round, or of two

struct Sides {
  uint64_t rows, cols;
};
// Two rounds at a time where the shorter side is so much shorter (see `operations_of`): then there are three symmetric matrices, else two.
inline bool in_pairs(uint64_t rows, uint64_t cols) { return std::max(rows, cols) >= 2 * std::min(rows, cols); }

// One product of the matrices of a shape: of X (from x[from]) with itself, of symmetric matrices s[left] s[right] that commute, or of s[left] and X; or all
// products of symmetric matrices of a round, or of two, from s[left] to s[out].
struct Operation {
  enum { kGram, kProduct, kMove, kChain, kChain2 } what;
  int left, right, out, add;                               // add: -1 for none
  float by, add_by, diagonal;
  bool last;
  bool chain() const { return what == kChain || what == kChain2; }
};
// A round by itself: G, P = a + b G + c G G, X <- P X.  Two rounds P' P X with the second one's G' = (P X)(P X)^T = P G P:
//   G, P, T = P G, G' = P T, P', Q = P' P, X <- Q X
// are five products of the shorter side alone in place of two products with X (work of 3 short^2 long for one of 3 short^3): 1024 x 4096 takes three quarters
// of the operations.  Not more rounds at a time: what rounding leaves in G for small singular values grows by a^2 in each further one.
inline std::vector<Operation> operations_of(const Sides& k, uint32_t steps, float a, float b, float c, bool chain) {
  std::vector<Operation> ops;
  auto product = [&](int l, int r, int out, float by) { ops.push_back(Operation{Operation::kProduct, l, r, out, -1, by, 0.f, 0.f, false}); };
  auto polynomial = [&](int g, int out) { ops.push_back(Operation{Operation::kProduct, g, g, out, g, c * (kP / (kG * kG)), b * (kP / kG), a * kP, false}); };
  for (uint32_t i = 0; i < steps;) {
    ops.push_back(Operation{Operation::kGram, 0, 0, 0, -1, kG / (kX * kX), 0.f, 0.f, false});
    const bool two = i + 1 < steps && in_pairs(k.rows, k.cols);
    if (chain) ops.push_back(Operation{two ? Operation::kChain2 : Operation::kChain, 0, 0, 1, -1, 0.f, 0.f, 0.f, false});
    else polynomial(0, 1);
    if (two && !chain) {
      product(1, 0, 2, 1.f / kP);                          // T as G: its eigenvalues are products of two singular values of X, before and after
      product(1, 2, 0, 1.f / kP);
      polynomial(0, 2);
      product(2, 1, 0, kQ / (kP * kP));
    }
    i += two ? 2 : 1;
    const float held = two ? kQ : kP;
    ops.push_back(Operation{Operation::kMove, two && !chain ? 0 : 1, 0, 0, -1, i < steps ? 1.f / held : 1.f / (held * kX), 0.f, 0.f, i == steps});
  }
  return ops;
}

// What one launch does: the next operation of every shape that has one left, by its place in the list.
struct Launch {
  std::vector<std::pair<size_t, Operation>> ops;
  bool chain = false;                                      // by the kernel for narrow matrices: then all shapes' operations are the same one
};
// The launches of a group of shapes, one behind the other.  The kernel for narrow matrices is taken where all of them are (beside larger matrices the products of
// narrow ones cost no launch of their own).  Those are far longer than wide, beyond what one CTA holds, and so all have the same operations; the others' lists differ in length.
inline std::vector<Launch> launches_of(const std::vector<Sides>& shapes, uint32_t steps, float a, float b, float c) {
  bool chain = true;
  for (const Sides& k : shapes) chain = chain && std::min(k.rows, k.cols) <= kNarrow;
  std::vector<std::vector<Operation>> ops;
  size_t most = 0;
  for (const Sides& k : shapes) {
    ops.push_back(operations_of(k, steps, a, b, c, chain));
    most = std::max(most, ops.back().size());
  }
  std::vector<Launch> launches(most);
  for (size_t i = 0; i < most; ++i) {
    for (size_t k = 0; k < shapes.size(); ++k)
      if (i < ops[k].size()) launches[i].ops.emplace_back(k, ops[k][i]);
    launches[i].chain = launches[i].ops[0].second.chain();   // (the first shape's list may have ended, the longest one has not)
  }
  return launches;
}

}  // namespace muon
}  // namespace polar_b200
