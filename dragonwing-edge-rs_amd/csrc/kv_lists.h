// What the lists of a paged cache say.  They live on the device and hold
// whatever their writer left there: nothing here overflows or leads out of the
// buffers, for any of an int's values.
#pragma once

namespace dw {

// New tokens [first, first + count) of a sequence that the list has from row t0
// up to row t1, of `tokens` rows.
struct NewTokens {
  int first, count;
};
__host__ __device__ __forceinline__ NewTokens new_tokens(int t0, int t1, int tokens) {
  const int first = t0 < 0 ? 0 : t0 < tokens ? t0 : tokens, end = t1 < 0 ? 0 : t1 < tokens ? t1 : tokens;
  return {first, end > first ? end - first : 0};
}

// Whether an entry of the joins' table (first slot, splits, first token, first
// head) can be followed.  Lists that overlap make more items than the splits
// that note them: an entry may then hold anything, and a head near an int's end
// would wrap as the rows' heads are counted from it.
__host__ __device__ __forceinline__ bool entry_fits(int slot, int splits, int token, int head, int slots, int tokens,
                                                    int heads) {
  return splits > 1 && slot >= 0 && slot <= slots - splits && token >= 0 && token < tokens && head >= 0 && head < heads;
}

}  // namespace dw
