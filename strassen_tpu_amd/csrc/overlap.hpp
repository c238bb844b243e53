// Which elements strided operands share: host checks of the serving operators,
// whose workgroups read and write them in no particular order.
#pragma once

#include <cstdint>

namespace smx {

// Runs of `width` bf16 values: up to three dimensions of them, strides in elements (not negative).
struct Runs {
  const void* at;
  int64_t width;
  struct {
    int64_t count, stride;
  } dims[3];

  // Its dimensions by stride, ascending; one of a single run is none.
  Runs sorted() const {
    Runs r = *this;
    for (auto& d : r.dims)
      if (d.count <= 1) d.count = 1, d.stride = 0;
    auto order = [&](int a, int b) {
      if (r.dims[a].stride > r.dims[b].stride) {
        const auto d = r.dims[a];
        r.dims[a] = r.dims[b], r.dims[b] = d;
      }
    };
    order(0, 1), order(1, 2), order(0, 1);
    return r;
  }
  // Elements from the first to behind the last.
  int64_t extent() const {
    int64_t e = width;
    for (const auto& d : dims)
      if (d.count > 1) e += (d.count - 1) * d.stride;
    return e;
  }
};

// Whether no two runs share an element: each dimension steps over all that the smaller strides span.
// (Layouts that interleave their dimensions otherwise are taken to overlap.)
inline bool lie_apart(const Runs& runs) {
  const Runs r = runs.sorted();
  int64_t span = r.width;
  for (const auto& d : r.dims) {
    if (d.count <= 1) continue;
    if (d.stride < span) return false;
    span += (d.count - 1) * d.stride;
  }
  return true;
}

// Whether a run of a shares an element with a run of b that lies `distance` elements behind it at the same
// indices, for operands of the same strides that lie apart: the distance less a sum of whole steps is below a run.
inline bool meet_at(const Runs& r, int dim, int64_t distance) {
  if (dim < 0) return distance > -r.width && distance < r.width;
  const auto& d = r.dims[dim];
  if (d.count <= 1) return meet_at(r, dim - 1, distance);
  int64_t steps = distance / d.stride;
  if (distance % d.stride < 0) --steps;
  for (int64_t s = steps; s <= steps + 1; ++s)
    if (s > -d.count && s < d.count && meet_at(r, dim - 1, distance - s * d.stride)) return true;
  return false;
}

// Whether two operands that lie apart each share elements: exact for the same shape and strides (parts of
// one tensor); others are taken to where the memory from their first to their last element does.
inline bool meet(const Runs& x, const Runs& y) {
  const Runs a = x.sorted(), b = y.sorted();
  const auto from_a = (intptr_t)a.at, from_b = (intptr_t)b.at;
  if (from_a + 2 * a.extent() <= from_b || from_b + 2 * b.extent() <= from_a) return false;
  bool alike = a.width == b.width && (from_b - from_a) % 2 == 0;
  for (int i = 0; i < 3; ++i) alike = alike && a.dims[i].count == b.dims[i].count && a.dims[i].stride == b.dims[i].stride;
  return !alike || !lie_apart(a) || meet_at(a, 2, (from_b - from_a) / 2);
}

// Whether `count` values from `list` on share memory with the rows of a table of `size`-byte values
// (rows at least `width` apart, from each first value on).
inline bool list_meets_table(const void* list, int64_t count, const void* table, int64_t rows, int64_t width,
                             int64_t stride, int64_t size) {
  const int64_t from = (intptr_t)list - (intptr_t)table, to = from + count * size, row = stride * size;
  if (count <= 0) return false;
  // the first row that ends behind the list's start
  const int64_t first = from < width * size ? 0 : (from - width * size) / row + 1;
  return first < rows && first * row < to;
}

// The same elements at the same indices.
inline bool same_runs(const Runs& x, const Runs& y) {
  bool same = x.at == y.at && x.width == y.width;
  for (int i = 0; i < 3; ++i)
    same = same && x.dims[i].count == y.dims[i].count && (x.dims[i].count <= 1 || x.dims[i].stride == y.dims[i].stride);
  return same;
}

}  // namespace smx
