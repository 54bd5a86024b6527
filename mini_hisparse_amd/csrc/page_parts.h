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

// A window shows a request's newest `window` tokens and its first `sinks`: those from `lo` on and
// those below `sinks`.  The whole tiles between them are passed over: of the tiles that are walked,
// those below `front` are the request's own, the others lie `gap` further on.
constexpr int32_t NO_WINDOW = 0x7fffffff;  // no request is longer

struct Seen {
  int32_t lo, front, gap;
};
__host__ __device__ __forceinline__ Seen seen_of(int32_t n, int32_t window, int32_t sinks) {
  const int32_t lo = n > window ? n - window : 0, first = lo / PM_TILE, front = tiles_of(sinks);
  return Seen{lo, front, first > front ? first - front : 0};
}
__host__ __device__ __forceinline__ int32_t seen_tiles(int32_t n, int32_t window, int32_t sinks) {
  return tiles_of(n) - seen_of(n, window, sinks).gap;
}
// The tokens (bits) of the tile from token `base` < lo on that are seen.
__host__ __device__ __forceinline__ uint32_t seen_mask(int32_t base, int32_t lo, int32_t sinks) {
  const int32_t before = lo - base, first = sinks - base;
  return (before < PM_TILE ? 0xffffffffu << before : 0u) |
         (first <= 0 ? 0u : (first < PM_TILE ? (1u << first) - 1u : 0xffffffffu));
}
// The most tokens, and tiles, that any request of up to `tokens` has to see (its window may begin
// inside a tile).
__host__ __device__ __forceinline__ int64_t most_seen(int64_t tokens, int32_t window, int32_t sinks) {
  const int64_t seen = static_cast<int64_t>(window) + sinks;
  return seen < tokens ? seen : tokens;
}
__host__ __device__ __forceinline__ int64_t most_seen_tiles(int64_t tokens, int32_t window, int32_t sinks) {
  const int64_t all = (tokens + PM_TILE - 1) / PM_TILE;
  const int64_t seen = (static_cast<int64_t>(window) + PM_TILE - 2) / PM_TILE + 1 + tiles_of(sinks);
  return seen < all ? seen : all;
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
