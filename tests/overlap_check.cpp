// Host check of csrc/overlap.hpp against every element's address: operands of up to three dimensions with
// small counts and strides, at every distance. Built and run by tests/test_serving_edges.py.
#include <cstdio>
#include <set>
#include <vector>

#include "../strassen_tpu_amd/csrc/overlap.hpp"

static uint16_t memory[4096];

static std::vector<const uint16_t*> elements(const smx::Runs& r) {
  std::vector<const uint16_t*> all;
  for (int64_t a = 0; a < r.dims[0].count; ++a)
    for (int64_t b = 0; b < r.dims[1].count; ++b)
      for (int64_t c = 0; c < r.dims[2].count; ++c)
        for (int64_t e = 0; e < r.width; ++e)
          all.push_back((const uint16_t*)r.at + a * r.dims[0].stride + b * r.dims[1].stride + c * r.dims[2].stride + e);
  return all;
}

int main() {
  const int64_t counts[][3] = {{1, 1, 1}, {3, 1, 1}, {3, 2, 1}, {1, 2, 3}, {2, 3, 2}, {4, 2, 1}};
  const int64_t strides[] = {0, 1, 2, 4, 6, 9, 12, 24};
  long layouts = 0, pairs = 0, apart_found = 0, meets = 0;
  for (const auto& n : counts)
    for (int64_t x : strides)
      for (int64_t y : strides)
        for (int64_t z : strides)
          for (int64_t width : {1, 2, 4}) {
            const smx::Runs a{memory + 512, width, {{n[0], x}, {n[1], y}, {n[2], z}}};
            const auto list = elements(a);
            const std::set<const uint16_t*> set(list.begin(), list.end());
            const bool apart = set.size() == list.size();
            ++layouts;
            if (smx::lie_apart(a)) {
              ++apart_found;
              if (!apart) return printf("taken to lie apart: %ld %ld %ld width %ld\n", x, y, z, width), 1;
            }
            if (!smx::same_runs(a, a)) return printf("not the same\n"), 1;
            for (int64_t d = -a.extent() - 1; d <= a.extent() + 1; ++d, ++pairs) {
              smx::Runs b = a;
              b.at = memory + 512 + d;
              bool met = false;
              for (const auto* e : elements(b)) met = met || set.count(e);
              const bool said = smx::meet(a, b);
              // never missed; exact where the operands lie apart
              if (said != met && (met || smx::lie_apart(a)))
                return printf("meet %d, not %d: %ld %ld %ld width %ld distance %ld\n", said, met, x, y, z, width, d), 1;
              if (d && smx::same_runs(a, b)) return printf("the same at a distance\n"), 1;
              meets += met;
            }
            // another layout in the same memory
            const smx::Runs other{memory + 512 + 40, width, {{2, 8}, {2, 16}, {1, 0}}};
            bool met = false;
            for (const auto* e : elements(other)) met = met || set.count(e);
            if (met && !smx::meet(a, other)) return printf("missed another layout\n"), 1;
          }
  // lists among the rows of tables
  for (int64_t rows = 1; rows <= 3; ++rows)
    for (int64_t width = 1; width <= 4; ++width)
      for (int64_t stride = width; stride <= width + 3; ++stride)
        for (int64_t count = 0; count <= 5; ++count)
          for (int64_t at = -8; at <= rows * stride + 2; ++at) {
            bool met = false;
            for (int64_t r = 0; r < rows; ++r)
              for (int64_t e = at; e < at + count; ++e) met = met || (e >= r * stride && e < r * stride + width);
            const auto* table = (const int32_t*)memory + 64;
            if (smx::list_meets_table(table + at, count, table, rows, width, stride, 4) != met)
              return printf("table of %ld rows of %ld, %ld apart, list of %ld at %ld\n", rows, width, stride, count, at), 1;
          }
  // the layouts of heads lie apart: rows of tokens, heads outside tokens, columns of a wider product, one run
  const int64_t heads[][4] = {{16, 512, 4, 128}, {16, 128, 4, 2048}, {16, 768, 4, 128}, {1, 0, 1, 0}, {1, 5, 4, 128}};
  for (const auto& h : heads)
    if (!smx::lie_apart({memory, 128, {{h[0], h[1]}, {h[2], h[3]}, {1, 0}}})) return printf("heads taken to overlap\n"), 1;
  if (smx::lie_apart({memory, 128, {{16, 512}, {8, 128}, {1, 0}}})) return printf("heads over the next token's\n"), 1;
  printf("ok: %ld layouts, %ld apart, %ld pairs, %ld meet\n", layouts, apart_found, pairs, meets);
  return 0;
}
