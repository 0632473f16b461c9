// Views of [B, heads, S, D] tensors: what the launchers check and compute about them on the host.
#pragma once
#include <cstdint>

namespace kcg {

// Strides in elements; the innermost is 1.
struct HeadView {
  const void* base;
  int B, H, S, D;
  int64_t sb, sh, sr;
};

// bytes from the first to one past the last element
inline unsigned long long head_view_extent(const HeadView& v, int elem_bytes) {
  return (static_cast<unsigned long long>(v.B - 1) * v.sb + static_cast<unsigned long long>(v.H - 1) * v.sh +
          static_cast<unsigned long long>(v.S - 1) * v.sr + v.D) * elem_bytes;
}

// The bytes of a view, for views_overlap: rows of `row` bytes, n[i] of them every s[i] bytes, the largest stride
// first; extents of one and strides of zero add none.
struct HeadRegion {
  uintptr_t lo;
  long long row, span;            // of one row; from the first to one past the last byte
  int dims;
  long long n[3], s[3];
  HeadRegion(const HeadView& v, int elem_bytes) : lo(reinterpret_cast<uintptr_t>(v.base)), dims(0) {
    row = static_cast<long long>(v.D) * elem_bytes;
    const long long ext[3] = {v.B, v.H, v.S}, str[3] = {v.sb, v.sh, v.sr};
    const __int128 most = __int128{1} << 60;
    __int128 end = row;
    for (int i = 0; i < 3; ++i) {
      if (ext[i] <= 1 || str[i] <= 0) continue;
      if (str[i] > static_cast<long long>(most >> 4)) {
        end = most + 1;
        break;
      }
      end += static_cast<__int128>(ext[i] - 1) * str[i] * elem_bytes;
      int at = dims++;
      for (; at > 0 && s[at - 1] < str[i] * elem_bytes; --at) n[at] = n[at - 1], s[at] = s[at - 1];
      n[at] = ext[i];
      s[at] = str[i] * elem_bytes;
    }
    // (no allocation is that long: such a view is refused elsewhere or never read to its end)
    if (end > most) dims = 0;
    span = end > most ? row : static_cast<long long>(end);
  }
};

// Whether two views share memory, as far as that can be told without walking their rows: equal bases, and overlapping
// ranges of views without gaps once the strides whose periods keep the members apart (batches, tokens, heads of a
// packed buffer) are taken out.  False also where neither this nor its opposite can be told.
inline bool views_overlap(HeadRegion a, HeadRegion b) {
  if (a.lo == b.lo) return true;
  long long d = static_cast<long long>(b.lo - a.lo);
  int i = 0, j = 0;      // strides taken out of a and of b
  for (;;) {
    if (d >= a.span || -d >= b.span) return false;
    if (i == a.dims && j == b.dims) return true;
    // the larger stride; one member of the view that does not have it
    const long long sa = i < a.dims ? a.s[i] : 0, sb = j < b.dims ? b.s[j] : 0, s = sa > sb ? sa : sb;
    const long long na = sa == s ? a.n[i] : 1, nb = sb == s ? b.n[j] : 1;
    // What is left without it, and where the first of b is in the period of a: r past its q-th member, or s - r
    // before the next.  If both stay inside one period, only members q apart can meet.
    const long long ra = a.span - (na - 1) * s, rb = b.span - (nb - 1) * s;
    long long q = d >= 0 ? d / s : -((-d + s - 1) / s), r = d - q * s;
    if (r + rb > s || ra > s) {
      if (s - r + ra > s || rb > s) break;
      ++q;
      r -= s;
    }
    if (q >= na || -q >= nb) return false;
    d = r;
    a.span = ra;
    b.span = rb;
    i += sa == s;
    j += sb == s;
  }
  auto gaps = [](const HeadRegion& v, int from) {
    long long filled = v.row;
    for (int k = v.dims - 1; k >= from; --k) {
      if (v.s[k] > filled) return true;
      filled += (v.n[k] - 1) * v.s[k];
    }
    return false;
  };
  return !gaps(a, i) && !gaps(b, j);
}

}  // namespace kcg
