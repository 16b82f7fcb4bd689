// The host rules for clusters, with devices that hold clusters of 16, of 8 only, or answer with an error.
#include <cstdio>

#include "mcpm_cluster.h"

int main() {
    int asked = 0;
    auto holds = [&](int most) { return [&asked, most](int width) { ++asked; return width <= most ? 4 : most < 0 ? -1 : 0; }; };
    const int got[] = {mcpm::widest_cluster(16, holds(16)), mcpm::widest_cluster(16, holds(8)), mcpm::widest_cluster(16, holds(-1)),
                       mcpm::widest_cluster(8, holds(0)), mcpm::widest_cluster(1, holds(0)), asked, mcpm::cluster_ctas(148),
                       mcpm::cluster_ctas(132), mcpm::cluster_ctas(7)};
    for (int x : got) std::printf("%d ", x);
    return 0;
}
