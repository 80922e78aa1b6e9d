// kv8_attend_e4m3.hip -- the attention kernels of the e4m3 cache (built apart for build time).
#include "kv8_attend.hpp"

namespace csahca {

int kv8_attend_launch_e4m3(const Kv8Attend& a, int tiles, hipStream_t stream) {
  return kv8_attend_launch<E4m3>(a, tiles, stream);
}

}  // namespace csahca
