// paged_tiles.hpp — how many tiles the query rows of a batch can make (host arithmetic of
// flash_attention_paged_prefix, whose lengths only the device knows).
#pragma once

#include <cstdint>
#include <numeric>

namespace nfhip {

// A batch's query rows of one KV head, `rows` in all, lie in at most `parts` parts, each of
// which has a multiple of `group` of them.  A part of up to `few` rows is cut into tiles of
// `narrow`, another into tiles of up to `wide`, a multiple of `narrow`.
//
// With g the common divisor of `group` and a tile height T, a part's rows r and T are
// multiples of g, so ceil(r / T) <= (r + T - g) / T.  All parts have no more tiles than
// those of `narrow`, (rows + parts (narrow - g)) / narrow; and where x <= min(rows, few
// parts) rows are in narrow tiles, no more than (rows - x) / wide + x / narrow + parts (1 -
// g / wide).
inline uint64_t most_tiles(uint64_t rows, uint64_t parts, uint64_t group, uint64_t few, uint64_t narrow, uint64_t wide) {
  if (parts > rows / group) parts = rows / group;  // with a row at all
  const uint64_t x = rows < few * parts ? rows : few * parts;
  const uint64_t a = (rows + parts * (narrow - std::gcd(group, narrow))) / narrow;
  const uint64_t b = (rows + (wide / narrow - 1) * x + parts * (wide - std::gcd(group, narrow))) / wide;
  return a < b ? a : b;
}

}  // namespace nfhip
