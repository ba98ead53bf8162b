// attend_shared.hip — attention over a cache of 16 bits with shared prefixes (mars_kv_attend_shared).
#include "attend.hpp"

namespace mars {

int launch_attend_shared(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s) { return launch_form<Shared>(r, a, max_new, s); }

}  // namespace mars
