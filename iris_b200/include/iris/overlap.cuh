// overlap.cuh — whether arrays share memory, for the checks of an entry point (host code).
//
// An array is rows of `bytes` bytes at up to three pitches.  Two rows meet where the difference of their places, a sum of
// multiples of the pitches, falls within a range; with pitches that nest (each as long as all rows within it) only two or three
// multiples of the largest come into question, for each of those of the next, and so on.
#pragma once
#include <stdint.h>

namespace iris {
namespace overlap {

struct Rows {
  const void* at;
  int64_t bytes;
  struct {
    int64_t n, pitch;      // pitch in bytes
  } dim[3];
};

inline Rows one_row(const void* at, int64_t bytes) { return {at, at ? bytes : 0, {{1, 0}, {1, 0}, {1, 0}}}; }
inline Rows matrix(const void* at, int64_t bytes, int64_t n, int64_t pitch) { return {at, at ? bytes : 0, {{n, pitch}, {1, 0}, {1, 0}}}; }

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

// Whether a and b share memory: exactly, if both are laid out alike or one is a single row (and the pitches nest); else whether the
// memory from the first to the last byte of the one meets that of the other.
inline bool meet(const Rows& a0, const Rows& b0) {
  if (a0.bytes <= 0 || b0.bytes <= 0) return false;
  const Rows a = sorted(a0), b = sorted(b0);
  int64_t a_span = a.bytes, b_span = b.bytes;
  bool alike = true, a_one = true, b_one = true;
  for (int i = 0; i < 3; ++i) {
    if (a.dim[i].n < 1 || b.dim[i].n < 1) return false;
    a_span += (a.dim[i].n - 1) * a.dim[i].pitch, b_span += (b.dim[i].n - 1) * b.dim[i].pitch;
    alike = alike && a.dim[i].n == b.dim[i].n && a.dim[i].pitch == b.dim[i].pitch;
    a_one = a_one && a.dim[i].n == 1, b_one = b_one && b.dim[i].n == 1;
  }
  const int64_t off = (int64_t)(reinterpret_cast<uintptr_t>(b.at) - reinterpret_cast<uintptr_t>(a.at));
  if (off >= a_span || off <= -b_span) return false;
  // a row of a at off_a and one of b at off + off_b meet if off - a.bytes < off_a - off_b < off + b.bytes
  if (b_one && apart(a)) return reaches(a, 0, 0, off - a.bytes, off + b.bytes);
  if (a_one && apart(b)) return reaches(b, 0, 0, -off - b.bytes, -off + a.bytes);
  if (alike && apart(a)) return reaches(a, 0, 1, off - a.bytes, off + b.bytes);
  return true;
}

}  // namespace overlap
}  // namespace iris
