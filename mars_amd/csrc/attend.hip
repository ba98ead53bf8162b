// attend.hip — attention over a cache of 16 bits (mars_kv_attend).
#include "attend.hpp"

namespace mars {

int launch_attend(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s) { return launch_form<Plain>(r, a, max_new, s); }

}  // namespace mars
