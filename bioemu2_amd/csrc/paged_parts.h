// Into parts of which length the keys of a paged attention call are cut (paged.hip): on the GPU, by the lengths there.
#pragma once

namespace bioemu {

#ifdef __HIPCC__
#define BIOEMU_DEVICE __device__ __forceinline__
#else
#define BIOEMU_DEVICE inline
#endif

// `total` tiles, `live` items that have some, `groups` workgroups at a time; parts(n): how many parts of up to n tiles
// there are (every item is cut into equal parts); search: whether that may be asked for more than once.
// The shortest parts that all run at once, to six tiles, if they are up to kMost tiles or a sixth longer than an equal
// share; else kLonger longer, and the last ones start late. Parts of `even` tiles leave a workgroup for the last part of
// every item, so they all run at once (where there are more workgroups than items): they are taken without a search where
// they are little longer than a share.
// 131072 and 118528 keys of 32 key heads of 64 in bf16: parts 24 tiles longer, 32 of 544 of which started late, took 379
// us; 26 longer, none of which does, 323. Four contexts of 48000 to 131072 keys, 16 key heads: 274 and 225.
// Measured in a graph, with such parts 16, 24 and 48 tiles longer: 48 sequences of up to 2000 keys, 8 key heads of 128,
// 51 us, 47 and 54; 32 of up to 2048, 34, 36 and 36; 100 of up to 3000, 4 key heads, 68, 65 and 65; 56 of up to 2000, 8
// key heads of 80, 42, 42 and 38: with 24 they take the least together.
constexpr unsigned kLonger = 24, kMost = 48;

template <class Parts>
BIOEMU_DEVICE unsigned part_length(unsigned total, unsigned live, unsigned groups, unsigned least, bool search,
                                   const Parts& parts) {
  const unsigned even = groups > live ? (total + groups - live - 1) / (groups - live) : ~0u, each = total / groups;
  const unsigned sixth = each / 6 + 4, few = sixth < kLonger ? sixth : kLonger;
  if (even <= each + few || even <= least) return even > least ? even : least;
  const unsigned near = search ? kMost : kLonger, most = each + (near > sixth ? near : sixth);
  if (!search) return even <= most ? even : each + kLonger;
  unsigned fits = most;
  if (parts(fits) > groups) return each + kLonger;
  for (unsigned less = each; fits - less > 6;) {
    const unsigned n = less + (fits - less) / 2;
    if (parts(n) <= groups) fits = n;
    else less = n;
  }
  return fits > least ? fits : least;
}

}  // namespace bioemu
