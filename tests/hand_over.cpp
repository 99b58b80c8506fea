// The hand-overs of attention's dq kernel (cswap_b200/csrc/attention_kernels.cu), every order of events: warps as lists of
// arrivals and waits on mbarriers, whose phases a wait tells by their parity alone, as the hardware's do.  A state in
// which nobody can go on and not all have ended is one in which the kernel's waits run out.
//
//   hand_over <turns>     turns: 3, both hand-overs on two barriers in turn (the kernel); 1 and 2, the rows' or the sums' on
//                         a single one.  Exits with 0 where every order comes to its end, 1 where one does not.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "../cswap_b200/csrc/hand_over.cuh"

namespace {

constexpr int kPieces = 5;
struct Op {
  bool wait;
  uint32_t bar, parity;
};
enum : uint32_t { kRows = 0, kLeft = 16, kScores = 32, kScoresFree = 40, kSlopes = 48, kGradients = 56, kFull = 64, kFree = 72,
                  kMeetResults = 80, kMeetSoftmax = 88, kEnd = 96 };

struct Model {
  std::vector<std::vector<Op>> warps;
  uint32_t count[kEnd / 8];
  std::set<std::vector<uint8_t>> seen;

  uint32_t arrivals(const std::vector<uint8_t>& at, uint32_t bar) const {
    uint32_t n = 0;
    for (size_t w = 0; w < warps.size(); ++w)
      for (int i = 0; i < at[w]; ++i) n += !warps[w][i].wait && warps[w][i].bar == bar;
    return n;
  }
  // a wait for a parity ends where the phase that runs has the other one
  bool open(const std::vector<uint8_t>& at, const Op& op) const {
    return !op.wait || (arrivals(at, op.bar) / count[op.bar / 8]) % 2 != op.parity;
  }
  bool all_end() {
    std::vector<std::vector<uint8_t>> todo{std::vector<uint8_t>(warps.size(), 0)};
    while (!todo.empty()) {
      const std::vector<uint8_t> at = todo.back();
      todo.pop_back();
      if (!seen.insert(at).second) continue;
      bool moved = false, ended = true;
      for (size_t w = 0; w < warps.size(); ++w) {
        if (at[w] == warps[w].size()) continue;
        ended = false;
        if (!open(at, warps[w][at[w]])) continue;
        moved = true;
        std::vector<uint8_t> then = at;
        ++then[w];
        todo.push_back(then);
      }
      if (!moved && !ended) return false;
    }
    return true;
  }
};

}  // namespace

int main(int argc, char** argv) {
  const int turns = argc > 1 ? std::atoi(argv[1]) : 3;
  auto bar = [&](uint32_t first, int which, uint32_t piece) { return turns & which ? csw::Turns{first}.bar(piece) : first; };
  auto parity = [&](int which, uint32_t piece) { return turns & which ? csw::Turns::parity(piece) : piece % 2; };
  Model m;
  for (uint32_t& c : m.count) c = 2;  // two warps stand for a group of them
  for (uint32_t b : {kScores, kSlopes, kFull}) m.count[b / 8] = 1;  // the products' own

  std::vector<Op> results, softmax, products;
  uint32_t met = 0;
  auto arrive = [](std::vector<Op>& w, uint32_t b) { w.push_back({false, b, 0}); };
  auto wait = [](std::vector<Op>& w, uint32_t b, uint32_t p) { w.push_back({true, b, p}); };
  auto finish = [&](uint32_t u) {
    wait(results, bar(kLeft, 2, u), parity(2, u));
    wait(results, kFull, u % 2);
    arrive(results, kFree);
    arrive(results, kMeetResults), wait(results, kMeetResults, met++ % 2);  // the staged tile is free, and full
  };
  for (uint32_t u = 0; u < kPieces; ++u) {
    arrive(results, kMeetResults), wait(results, kMeetResults, met++ % 2);
    arrive(results, bar(kRows, 1, u));
    if (u > 0) finish(u - 1);

    wait(softmax, bar(kRows, 1, u), parity(1, u));
    arrive(softmax, kMeetSoftmax), wait(softmax, kMeetSoftmax, u % 2);
    wait(softmax, kScores, u % 2);
    arrive(softmax, kScoresFree);
    wait(softmax, kSlopes, u % 2);
    arrive(softmax, kGradients);
    arrive(softmax, bar(kLeft, 2, u));

    if (u > 0) wait(products, kScoresFree, (u - 1) % 2);
    arrive(products, kScores), arrive(products, kSlopes);
    if (u > 0) wait(products, kFree, (u - 1) % 2);
    wait(products, kGradients, u % 2);
    arrive(products, kFull);
  }
  finish(kPieces - 1);
  m.warps = {results, results, softmax, softmax, products};
  const bool ok = m.all_end();
  std::printf("%zu states, %s\n", m.seen.size(), ok ? "all orders end" : "an order does not end");
  return ok ? 0 : 1;
}
