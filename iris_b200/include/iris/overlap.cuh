// overlap.cuh — whether arrays share memory, for the checks of an entry point (host code).
//
// An array is rows of `bytes` bytes at up to three pitches.  Two rows meet where the difference of their places, a sum of
// multiples of the pitches, falls within a range; with pitches that nest (each as long as all rows within it) only two or three
// multiples of the largest come into question, for each of those of the next, and so on.
#pragma once
#include <stdint.h>

namespace iris {
namespace overlap {

struct Dim {
  int64_t n, pitch;        // pitch in bytes
};
struct Rows {
  uintptr_t at, end;       // first byte, and the one behind the last
  int64_t bytes;
  Dim dim[3];
  Rows(const void* p, int64_t row, Dim a = {1, 0}, Dim b = {1, 0}, Dim c = {1, 0})
      : at(reinterpret_cast<uintptr_t>(p)), bytes(p ? row : 0), dim{a, b, c} {
    end = at;
    if (bytes > 0 && a.n > 0 && b.n > 0 && c.n > 0) end += bytes + (a.n - 1) * a.pitch + (b.n - 1) * b.pitch + (c.n - 1) * c.pitch;
  }
};

// The dimensions of more than one, largest pitch first.
inline Rows sorted(Rows r) {
  for (auto& d : r.dim)
    if (d.n == 1) d.pitch = 0;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (r.dim[j].pitch < r.dim[j + 1].pitch) {
        const auto d = r.dim[j];
        r.dim[j] = r.dim[j + 1], r.dim[j + 1] = d;
      }
  return r;
}

// Whether the pitches nest, so that no two rows share memory.
inline bool apart(const Rows& rows) {
  const Rows r = sorted(rows);
  int64_t need = r.bytes;
  for (int i = 2; i >= 0; --i) {
    if (r.dim[i].n <= 1) continue;
    if (r.dim[i].pitch < need) return false;
    need += (r.dim[i].n - 1) * r.dim[i].pitch;
  }
  return true;
}

// Whether a sum of d_i * pitch_i with -back <= d_i / (n_i - 1) <= 1, from dimension i on, lies between lo and hi (not included).
inline bool reaches(const Rows& r, int i, int back, int64_t lo, int64_t hi) {
  if (i == 3 || r.dim[i].n <= 1) return lo < 0 && 0 < hi;
  int64_t rest = 0;        // the largest sum of the dimensions behind
  for (int k = i + 1; k < 3; ++k) rest += (r.dim[k].n > 1 ? r.dim[k].n - 1 : 0) * r.dim[k].pitch;
  const int64_t pitch = r.dim[i].pitch, most = r.dim[i].n - 1;
  int64_t from = (lo - rest) / pitch - 1, to = (hi + back * rest) / pitch + 1;
  if (from < -back * most) from = -back * most;
  if (to > most) to = most;
  for (int64_t d = from; d <= to; ++d)
    if (reaches(r, i + 1, back, lo - d * pitch, hi - d * pitch)) return true;
  return false;
}

inline bool meet_within(const Rows& a0, const Rows& b0) {   // (those whose first to last bytes meet)
  const int64_t off = (int64_t)(b0.at - a0.at);
  const Rows a = sorted(a0), b = sorted(b0);
  bool alike = true, a_one = true, b_one = true;
  for (int i = 0; i < 3; ++i) {
    alike = alike && a.dim[i].n == b.dim[i].n && a.dim[i].pitch == b.dim[i].pitch;
    a_one = a_one && a.dim[i].n == 1, b_one = b_one && b.dim[i].n == 1;
  }
  // a row of a at off_a and one of b at off + off_b meet if off - a.bytes < off_a - off_b < off + b.bytes
  if (b_one && apart(a)) return reaches(a, 0, 0, off - a.bytes, off + b.bytes);
  if (a_one && apart(b)) return reaches(b, 0, 0, -off - b.bytes, -off + a.bytes);
  if (alike && apart(a)) return reaches(a, 0, 1, off - a.bytes, off + b.bytes);
  return true;
}
// Whether a and b share memory: exactly, if both are laid out alike or one is a single row (and the pitches nest); else whether the
// memory from the first to the last byte of the one meets that of the other.
inline bool meet(const Rows& a, const Rows& b) { return a.at < b.end && b.at < a.end && a.at < a.end && b.at < b.end && meet_within(a, b); }

}  // namespace overlap
}  // namespace iris
