// CPU-only checks of the launch plans in host_util.h, compiled by tests/test_cpp_plan.py.
#include "host_util.h"

using hfk::join_warps;
constexpr int kResident = 148 * hfk::kJoinWarpsPerSm;
static_assert(join_warps(1, kResident) == 16 && join_warps(kResident / 16, kResident) == 16, "few rows");
static_assert(join_warps(kResident / 16 + 1, kResident) == 4 && join_warps(kResident / 4, kResident) == 4, "");
static_assert(join_warps(kResident / 4 + 1, kResident) == 2 && join_warps(kResident / 2, kResident) == 2, "");
static_assert(join_warps(kResident / 2 + 1, kResident) == 1, "");
static_assert(join_warps(1 << 27, kResident) == 1 && join_warps(1 << 28, kResident) == 1 && join_warps(1 << 30, kResident) == 1, "2^31 warps and more");

using hfk::write_wide;
static_assert(!write_wide(1, 128, true, false) && !write_wide((1 << 14) - 1, 128, false, false) && write_wide(1 << 14, 128, false, false), "");
static_assert(write_wide(1 << 14, 96, true, true) && write_wide(0x7fffffffll, 256, true, true), "rotated rows, whatever the cache");
static_assert(!write_wide(1 << 14, 64, true, false) && write_wide(1 << 16, 64, true, false) && write_wide(1 << 16, 16, false, false), "small heads");
static_assert(!write_wide(0x7fffffffll, 128, false, true) && !write_wide(1 << 20, 64, false, true), "copies never");

int main() { return 0; }
