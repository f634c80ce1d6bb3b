// How many pieces of the vocabulary a backward call of (rows, vocabulary, width) on a device of so many SMs has, and the entries of one.
#include "stg_head_plan.h"

#include <cstdio>
#include <cstdlib>

int main(int argc, char **argv)
{
    if (argc != 5) return 2;
    const stg::HeadPlan p = stg::head_shape(std::atoi(argv[1]), std::atoi(argv[2]), std::atoi(argv[3]), std::atoi(argv[4]), true);
    std::printf("%d %d\n", p.pieces, p.piece);
    return 0;
}
