// The token range of one group of a K-grouped product, cut off at the rows that the operands have.  The arithmetic needs
// no device: it is plain C++ once the three qualifiers below have a meaning.
#pragma once

namespace b200 {

struct TokenSpan {
  long long start, tokens;
  bool cut;   // the group named rows that do not exist
};

// `size` tokens from row `start` of `total`; any value of `size` (a negative one counts as zero) and 0 <= start <= total.
// No group reaches past `total`, so the sum over the groups cannot overflow either, and a bad size costs no more
// k-blocks than there are rows.
__host__ __device__ __forceinline__ TokenSpan span_of_size(long long start, long long size, long long total) {
  TokenSpan s;
  const long long room = total - start;
  s.start = start;
  s.cut = size > room;
  s.tokens = size < 0 ? 0 : s.cut ? room : size;
  return s;
}

// rows [start, end) of `total` from explicit bounds of any value; end <= start is an empty group
__host__ __device__ __forceinline__ TokenSpan span_of_bounds(long long start, long long end, long long total) {
  TokenSpan s;
  const long long lo = start < 0 ? 0 : start > total ? total : start;
  const long long hi = end > total ? total : end;
  s.start = lo;
  s.tokens = hi > lo ? hi - lo : 0;
  s.cut = end > start && s.tokens != end - start;
  return s;
}

}  // namespace b200
