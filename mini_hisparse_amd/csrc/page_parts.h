// Arithmetic of the attention over page tables' schedule (pages.hip): tiles of a request, and
// the size of the parts that all requests together are cut into.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hs {

constexpr int PM_TILE = 32;  // tokens

// A request's tokens, at most `limit`, and their tiles.
__host__ __device__ __forceinline__ int32_t clamp_length(int64_t n, int64_t limit) {
  return static_cast<int32_t>(n < 0 ? 0 : (n < limit ? n : limit));
}
__host__ __device__ __forceinline__ int32_t tiles_of(int32_t n) {
  return static_cast<int32_t>((static_cast<uint32_t>(n) + PM_TILE - 1) / PM_TILE);
}

// Parts are of `per` tiles, and an empty request has one.  All requests together are to need at
// most `target` workgroups: with per = sum n_b / (target - B) they surely do (sum ceil(n_b / per)
// <= sum n_b / per + B), but with sum n_b / target they may, as equal lengths often do.  The first
// of PM_TRIES sizes from this one up to the sure one that does is taken, where B is above a quarter
// of the target (fewer leave three quarters of the CUs busy in any case, and the search costs 1 us).
// In us without and with the smaller sizes: 64 requests of 16384, 40 query and 8 KV heads of 128
// in e4m3, 526 and 389; 128 of 4096, 28 and 4 heads in int8, 126 and 118.
constexpr int PM_TRIES = 4;

__host__ __device__ __forceinline__ uint32_t sure_room(int64_t target, int64_t B) {
  return static_cast<uint32_t>(target - (B < target / 2 ? B : target / 2));
}
// The sure size for `total` tiles.  Where B is well above the target, total / room may pass 32 bits
// (65535 requests of 2^31 tokens over a room of 256); no request has more than PM_MOST tiles, so no
// larger size is needed.
constexpr int64_t PM_MOST = int64_t{1} << 26;

__host__ __device__ __forceinline__ uint32_t sure_size(int64_t total, uint32_t room) {
  const int64_t size = (total + room - 1) / room;
  return static_cast<uint32_t>(size < PM_MOST ? size : PM_MOST);
}
// The same of a sum in fp32, which is exact below 2^24 tiles; above, more than its roundings can
// have lost is added.
__host__ __device__ __forceinline__ uint32_t sure_size(float total, uint32_t room) {
  if (total < 0x1p24f) return (static_cast<uint32_t>(total) + room - 1) / room;
  const float size = total / static_cast<float>(room) * 1.0001f;
  return size < static_cast<float>(PM_MOST) ? static_cast<uint32_t>(size) + 1u : static_cast<uint32_t>(PM_MOST);
}
__host__ __device__ __forceinline__ uint32_t tried_size(uint32_t least, uint32_t sure, int k, uint32_t min_tiles) {
  const uint32_t per = least + static_cast<uint32_t>(static_cast<uint64_t>(sure - least) * k / PM_TRIES);
  return per < min_tiles ? min_tiles : per;
}
__host__ __device__ __forceinline__ int32_t parts_of(int32_t tiles, uint32_t per) {
  return tiles > static_cast<int64_t>(per) ? static_cast<int32_t>((static_cast<uint32_t>(tiles) + per - 1) / per) : 1;
}

}  // namespace hs
