// Which lane of a warp copies which 16 bytes of the scales of a tile of a 4-bit
// cache, and where to. Plain C++, so that a program on the host can go through
// all lanes.
#pragma once

#ifdef __CUDACC__
#define LUNARA_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LUNARA_HOST_DEVICE inline
#endif

namespace lunara {

struct ScaleCopy {
  int kv, group, piece;   // 0 keys / 1 values, group of 8 keys of the tile, 16-byte piece of the group's scales
  int place;              // byte offset in the keys' or the values' scales of a stage
  bool copies;            // false: the lane has nothing to copy
};

// KT keys per tile, DP the head dimension rounded up, srow = head dimension / 16
// the scale bytes of a key. A group's scales are 8 * srow bytes, one group right
// behind the other. DP gives the lanes; those whose piece is beyond the group's
// bytes (srow < DP / 16) copy nothing: their place is the next group's, which
// another lane writes, and a copy that reads nothing writes zeros.
template <int KT, int DP>
LUNARA_HOST_DEVICE ScaleCopy scale_copy(int lane, int srow) {
  constexpr int kPieces = DP / 32, kLanes = (KT / 8) * kPieces;   // of the keys, and of the values
  const int rest = lane % kLanes, group = rest / kPieces, piece = rest % kPieces;
  return {lane / kLanes, group, piece, group * (8 * srow) + 16 * piece, lane < 2 * kLanes && 2 * piece < srow};
}

}  // namespace lunara
