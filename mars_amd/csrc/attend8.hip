// attend8.hip — attention over a cache of 8 bits, with or without shared prefixes (mars_kv_attend8).
#include "attend.hpp"

namespace mars {

int launch_attend8(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s) { return launch_form<Held8>(r, a, max_new, s); }

}  // namespace mars
