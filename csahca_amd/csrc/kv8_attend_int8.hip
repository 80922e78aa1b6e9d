// kv8_attend_int8.hip -- the attention kernels of the int8 cache (built apart for build time).
#include "kv8_attend.hpp"

namespace csahca {

int kv8_attend_launch_int8(const Kv8Attend& a, int tiles, hipStream_t stream) {
  return kv8_attend_launch<Int8>(a, tiles, stream);
}

}  // namespace csahca
