// Host-side check of the step from a row of Y, Z and the residual to a later one (csrc/fc_mma.cuh), for every pitch that a call may have.
#include <cstdio>
#include "../dragon-alpha-v1.0_b200/csrc/fc_mma.cuh"

int main()
{
    int bad = 0;
    for (int cols : {8, 4096, (1 << 28) - 8, 1 << 28, (1 << 28) + 8, 1 << 29, 1 << 30, 2147483647 - 1023})
        for (int rows : {1, 8, 24, 127}) {
            const unsigned long long want = static_cast<unsigned long long>(rows) * static_cast<unsigned>(cols);
            bad += alpha::fc_rows_on(rows, cols) != want;
            bad += alpha::fc_rows_on(rows, 2 * static_cast<size_t>(cols)) != 2 * want;
        }
    printf("%d wrong\n", bad);
    return bad != 0;
}
