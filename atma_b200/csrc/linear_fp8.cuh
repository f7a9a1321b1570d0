// Reads and clears the status word of the products in 8 bits (non-zero: a bounded wait ran out).
#pragma once

namespace atma {
int linear_fp8_status_fetch_and_clear(int* out);
}
