// The range of 64-bit keys in which the k-th largest of a list is looked for (csrc/top_logits.cu).
//
// The range is cut into up to 256 bins of 2^wide keys; the bin that holds the k-th largest is the next range, until what
// reaches its lower end is little more than k.  Keys above the bin are among the k already and must not be counted again.
// (No CUDA in here: the CPU tests compile it with a plain loop in the place of a block.)
#pragma once

#ifdef __CUDACC__
#define MMT_RANGE_FN __device__ __forceinline__
#else
#define MMT_RANGE_FN inline
#endif

struct KeyRange {
  static constexpr int kBins = 256;
  unsigned long long low, span;       // first key, and how far behind it the last one is
  int wide;

  // Keys whose bits from `shift` up are between `least` and `most`, both of 16 bits.
  MMT_RANGE_FN KeyRange(unsigned least, unsigned most, int shift)
      : low((unsigned long long)least << shift), span(~0ull), wide(shift) {
    while ((most - least) >> (wide - shift) >= (unsigned)kBins) ++wide;
  }
  MMT_RANGE_FN bool holds(unsigned long long key) const { return key >= low && key - low <= span; }
  // Of a key that the range holds.
  MMT_RANGE_FN int bin(unsigned long long key) const { return (int)((key - low) >> wide); }
  // On to the lower end of a bin, whose keys and those above are all that is left.
  MMT_RANGE_FN void raise(int to_bin) { low += (unsigned long long)to_bin << wide; }
  // The range is that bin, if its keys can be told apart.  A bin of fewer than 256 keys has as many bins, not 256.
  MMT_RANGE_FN bool narrow() {
    if (wide == 0) return false;
    span = (1ull << wide) - 1;
    wide = wide > 8 ? wide - 8 : 0;
    return true;
  }
};
