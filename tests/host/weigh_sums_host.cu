// The end of a block of tiles of the received weights, run by the host one thread of the block after the other.
#include "../../tenzo_b200/csrc/weigh_sums.cuh"

extern "C" void weigh_add_host(int groups, int given_up, int n, int t0, int t1, int total, const int* rows, const float* sums, float* weight) {
    if (groups == 3)
        for (int tid = 0; tid < 384; ++tid) tz::weigh_add<3, 42, 50, 384, 128, 16>(given_up != 0, tid, n, t0, t1, total, rows, sums, weight);
    else
        for (int tid = 0; tid < 512; ++tid) tz::weigh_add<4, 32, 40, 512, 128, 16>(given_up != 0, tid, n, t0, t1, total, rows, sums, weight);
}
