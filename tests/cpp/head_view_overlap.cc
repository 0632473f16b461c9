// views_overlap against the bytes themselves, for random small views: a "true" has to be true, and for views laid
// out as programs lay them out a "false" has to be false.  Prints how many of each there were.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>

#include "../../kernelcodegen_b200/csrc/head_view.h"

using kcg::HeadRegion;
using kcg::HeadView;

namespace {

std::mt19937 rng(1);
int pick(int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); }

std::set<long long> bytes(const HeadView& v, int es) {
  std::set<long long> all;
  const long long at = static_cast<long long>(reinterpret_cast<uintptr_t>(v.base));
  for (int b = 0; b < v.B; ++b)
    for (int h = 0; h < v.H; ++h)
      for (int s = 0; s < v.S; ++s)
        for (int i = 0; i < v.D * es; ++i) all.insert(at + (b * v.sb + h * v.sh + s * v.sr) * es + i);
  return all;
}

bool meet(const HeadView& a, int ea, const HeadView& b, int eb) {
  const std::set<long long> x = bytes(a, ea);
  for (const long long i : bytes(b, eb))
    if (x.count(i)) return true;
  return false;
}

const void* at(long long elements, int es) { return reinterpret_cast<const void*>(static_cast<uintptr_t>(4096 + elements * es)); }

// A view of some heads (and tokens) of a buffer of `total` heads, in one of the layouts in use.
HeadView part(int layout, int B, int S, int total, int D, int h0, int H, int s0, int s, int es) {
  switch (layout) {
    case 0: return {at((s0 * total + h0) * D, es), B, H, s, D, static_cast<int64_t>(S) * total * D, D, static_cast<int64_t>(total) * D};
    case 1: return {at((h0 * S + s0) * D, es), B, H, s, D, static_cast<int64_t>(S) * total * D, static_cast<int64_t>(S) * D, D};
    case 2: return {at((h0 * B * S + s0) * D, es), B, H, s, D, static_cast<int64_t>(S) * D, static_cast<int64_t>(B) * S * D, D};
    default: return {at((h0 * S + s0) * D, es), B, H, s, D, static_cast<int64_t>(S) * total * D, 2 * static_cast<int64_t>(S) * D, D};  // every second head
  }
}

}  // namespace

int main() {
  long long yes = 0, no = 0, untold = 0, wrong = 0;
  for (int i = 0; i < 60000; ++i) {      // anything
    HeadView v[2];
    int es[2];
    for (int k = 0; k < 2; ++k) {
      es[k] = pick(0, 1) ? 2 : 4;
      v[k] = {reinterpret_cast<const void*>(static_cast<uintptr_t>(4096 + 4 * pick(0, 60))), pick(1, 3), pick(1, 3), pick(1, 4), pick(1, 4),
              pick(0, 30), pick(0, 12), pick(0, 8)};
    }
    if (pick(0, 1)) v[1].sb = v[0].sb, v[1].sh = v[0].sh, es[1] = es[0];
    if (pick(0, 1)) v[1].sr = v[0].sr;
    const bool said = kcg::views_overlap(HeadRegion(v[0], es[0]), HeadRegion(v[1], es[1]));
    const bool is = meet(v[0], es[0], v[1], es[1]);
    if (said && !is) ++wrong;
    if (!said && is) ++untold;
    ++(said ? yes : no);
  }
  std::printf("%lld %lld %lld %lld\n", yes, no, untold, wrong);
  yes = no = untold = wrong = 0;
  for (int i = 0; i < 40000; ++i) {      // heads and tokens of one buffer
    const int layout = pick(0, 3), B = pick(1, 3), S = pick(1, 6), total = pick(2, 8), D = pick(1, 4), es = pick(0, 1) ? 2 : 4;
    HeadView v[2];
    for (int k = 0; k < 2; ++k) {
      const int step = layout == 3 ? 2 : 1, h0 = pick(0, total - 1), H = pick(1, (total - 1 - h0) / step + 1);
      const int s0 = pick(0, S - 1), s = pick(1, S - s0);
      v[k] = part(layout, B, S, total, D, h0, H, s0, s, es);
    }
    const bool said = kcg::views_overlap(HeadRegion(v[0], es), HeadRegion(v[1], es));
    const bool is = meet(v[0], es, v[1], es);
    if (said && !is) ++wrong;
    if (!said && is) ++untold;
    ++(said ? yes : no);
  }
  std::printf("%lld %lld %lld %lld\n", yes, no, untold, wrong);
  return 0;
}
