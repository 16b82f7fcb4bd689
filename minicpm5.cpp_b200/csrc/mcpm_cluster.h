// Host rules for kernels on thread-block clusters.
#pragma once

namespace mcpm {

// CTAs that such a kernel spreads over at most, one to an SM: an eighth of the SMs are left, since a cluster lies in
// one GPC and the GPCs' odd SMs hold none.
inline int cluster_ctas(int n_sm) { return n_sm - n_sm / 8; }

// The widest cluster, at most `want` CTAs (a power of two), that the device can run.  Eight are portable; more are
// asked for (active(width): how many such clusters can run at once, negative on an error).
template <typename Active>
int widest_cluster(int want, Active active) {
    int width = want;
    while (width > 8 && active(width) < 1) width /= 2;
    return width;
}

}  // namespace mcpm
