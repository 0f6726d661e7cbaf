// The entry points of decoding over a bounded cache with their arguments in one array: a Python call of 28 arguments takes
// 3.3 us by ctypes, packing them and passing one pointer 0.7 us, and small calls are bound by that.
#include <cstring>

#include "common.cuh"

using namespace im;

extern "C" int im_bounded_call(const void* words, size_t bytes) {
  clear_error();
  constexpr size_t MOST = 32;
  static const size_t counts[] = {20, 25, 29, 25, 17};  // words of each entry, its number and stream with them
  int64_t w[MOST];
  IM_REQUIRE(words && bytes >= sizeof(int64_t) && bytes <= sizeof(w) && bytes % sizeof(int64_t) == 0, IM_INVALID,
             "im_bounded_call: %zu bytes", bytes);
  memcpy(w, words, bytes);
  IM_REQUIRE(w[0] >= 0 && w[0] < (int64_t)(sizeof(counts) / sizeof(counts[0])) &&
                 bytes == counts[w[0]] * sizeof(int64_t),
             IM_INVALID, "im_bounded_call: entry %lld with %zu bytes", (long long)w[0], bytes);
  auto p = [&](int i) { return reinterpret_cast<void*>(w[i]); };
  auto i32 = [&](int i) { return reinterpret_cast<int32_t*>(w[i]); };
  auto f32 = [&](int i) { return reinterpret_cast<float*>(w[i]); };
  auto number = [&](int i) {
    double x;
    memcpy(&x, &w[i], sizeof(x));
    return x;
  };
  // types, layouts and flags: what an int does not hold is refused as -1 is
  auto flag = [&](int i) { return w[i] >= 0 && w[i] < (1 << 30) ? (int)w[i] : -1; };
  switch (w[0]) {
    case IM_CALL_ROPE:
      return im_rope(p(1), w[2], w[3], p(4), flag(5), p(6), flag(7), w[8], number(9), flag(10), flag(11), w[12], w[13],
                     w[14], flag(15), p(16), w[17], w[18], p(19));
    case IM_CALL_ROPE_KV:
      return im_rope_kv(p(1), p(2), flag(3), w[4], number(5), flag(6), i32(7), i32(8), i32(9), i32(10), w[11], w[12],
                        w[13], w[14], w[15], w[16], w[17], flag(18), p(19), p(20), p(21), i32(22), w[23], p(24));
    case IM_CALL_ATTENTION_WEIGHTS:
      return im_attention_weights(p(1), p(2), p(3), flag(4), i32(5), w[6], w[7], w[8], i32(9), i32(10), i32(11), w[12],
                                  w[13], w[14], w[15], w[16], w[17], w[18], w[19], w[20], (float)number(21), f32(22),
                                  f32(23), w[24], p(25), p(26), (size_t)w[27], p(28));
    case IM_CALL_CACHE_EVICT:
      return im_cache_evict(p(1), p(2), w[3], w[4], w[5], i32(6), w[7], i32(8), i32(9), f32(10), f32(11), i32(12),
                            i32(13), i32(14), w[15], w[16], w[17], w[18], w[19], w[20], w[21], p(22), (size_t)w[23],
                            p(24));
    default:
      return im_verify_sampled(p(1), w[2], p(3), w[4], flag(5), i32(6), w[7], i32(8), f32(9), w[10], w[11], w[12],
                               w[13], i32(14), i32(15), p(16));
  }
}
