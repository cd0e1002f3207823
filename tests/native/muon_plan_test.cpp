// Host-side check of the order of orthogonalised momentum's products (csrc/muon_plan.hpp), the code that the step itself runs: for lists of
// shapes in every mixture every operation of every shape is launched once and in its order, the kernel for narrow matrices gets nothing but
// narrow ones, and nothing beyond a list's end is read (built with the address sanitizer).
#include <muon_plan.hpp>

#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace polar_b200::muon;

static int failures = 0, checked = 0;
#define CHECK(cond)                                                   \
  do {                                                                \
    if (!(cond)) {                                                    \
      if (failures < 20) std::printf("FAIL line %d: %s\n", __LINE__, #cond); \
      ++failures;                                                     \
    }                                                                 \
  } while (0)

static bool same(const Operation& a, const Operation& b) {
  return a.what == b.what && a.left == b.left && a.right == b.right && a.out == b.out && a.add == b.add && a.by == b.by && a.add_by == b.add_by &&
         a.diagonal == b.diagonal && a.last == b.last;
}

static void check(const std::vector<Sides>& shapes, uint32_t steps) {
  const float a = 3.4445f, b = -4.7750f, c = 2.0315f;
  bool narrow = true;
  for (const Sides& s : shapes) narrow = narrow && std::min(s.rows, s.cols) <= 128;
  std::vector<size_t> done(shapes.size(), 0);
  std::vector<std::vector<Operation>> want;
  for (const Sides& s : shapes) want.push_back(operations_of(s, steps, a, b, c, narrow));
  for (const Launch& l : launches_of(shapes, steps, a, b, c)) {
    CHECK(!l.ops.empty());
    CHECK(!l.chain || narrow);
    if (l.chain) CHECK(l.ops.size() == shapes.size());
    for (const auto& o : l.ops) {
      CHECK(o.first < shapes.size());
      CHECK(o.second.chain() == l.chain);
      CHECK(!l.chain || o.second.what == l.ops[0].second.what);
      CHECK(done[o.first] < want[o.first].size() && same(o.second, want[o.first][done[o.first]]));
      ++done[o.first];
    }
  }
  for (size_t k = 0; k < shapes.size(); ++k) {
    CHECK(done[k] == want[k].size());                      // every operation, once
    CHECK(want[k].back().what == Operation::kMove && want[k].back().last);
    uint32_t rounds = 0;                                   // and they are the rounds that were asked for
    for (size_t i = 0; i < want[k].size(); ++i) {
      if (want[k][i].what != Operation::kGram) continue;
      size_t n = 1;
      while (i + n < want[k].size() && want[k][i + n].what != Operation::kGram) ++n;
      const bool two = narrow ? want[k][i + 1].what == Operation::kChain2 : n == 7;
      CHECK(n == (narrow ? 3u : two ? 7u : 3u));
      rounds += two ? 2 : 1;
    }
    CHECK(rounds == steps);
  }
  ++checked;
}

int main() {
  // sides within a factor of two have lists of 3 operations a round, the others of 7 for two rounds: the longer list may stand anywhere
  const std::vector<Sides> near = {{1511, 777}, {999, 601}, {1024, 1024}, {301, 514}, {130, 140}, {4096, 4096}};
  const std::vector<Sides> far = {{999, 301}, {512, 1024}, {4096, 10}, {784, 4096}, {300, 150}};
  const std::vector<Sides> narrow = {{128, 2000}, {8192, 32}, {1, 16384}, {600, 9}, {4, 3000}};
  for (uint32_t steps : {1, 2, 3, 4, 5, 6, 7, 8, 31, 32}) {
    check({{1511, 777}, {999, 301}, {301, 514}}, steps);
    check({{1024, 1024}, {512, 1024}}, steps);
    for (const auto* one : {&near, &far, &narrow}) {
      for (const Sides& s : *one) check({s}, steps);
      check(*one, steps);
      for (const auto* other : {&near, &far, &narrow})
        for (const Sides& s : *one)
          for (const Sides& t : *other) check({s, t}, steps), check({t, t, s}, steps);
    }
    for (int i = 0; i < 200; ++i) {
      std::vector<Sides> shapes;
      for (int n = 1 + std::rand() % 20; n > 0; --n) shapes.push_back(Sides{129 + (uint64_t)std::rand() % 2000, 129 + (uint64_t)std::rand() % 2000});
      check(shapes, steps);
    }
  }
  std::printf("%d lists, %d failures\n", checked, failures);
  return failures != 0;
}
