// Driver in the style of the reference's *-run-fpga.cpp programs for gemm_grouped(OpB, X, W, Offsets, Y) and its matrix
// gradient: build buffers, call, re-check every output with a naive loop.
#include "gemm_grouped-interface.h"
#include "driver_common.h"

int main() {
    const int T = 100, E = 4, K = 40, N = 30;
    const int off[E + 1] = {3, 40, 40, 41, 96};
    t2sp::Buffer<float> x(K, T), w(N, K, E), y(N, T), dy(N, T), dw(N, K, E);
    t2sp::Buffer<int32_t> offsets(E + 1);
    drv::Rng rx(51), rw(52), ry(53);
    for (int t = 0; t < T; t++)
        for (int k = 0; k < K; k++) x(k, t) = rx.next();
    for (int e = 0; e < E; e++)
        for (int k = 0; k < K; k++)
            for (int n = 0; n < N; n++) w(n, k, e) = rw.next();
    for (int t = 0; t < T; t++)
        for (int n = 0; n < N; n++) { dy(n, t) = ry.next(); y(n, t) = 7.0f; }
    for (int e = 0; e <= E; e++) offsets(e) = off[e];
    if (int err = gemm_grouped(0, x, w, offsets, y)) { std::printf("gemm_grouped returned %d\n", err); return 1; }
    const double ns = t2sp_last_kernel_ns();
    if (int err = gemm_grouped_wgrad(x, dy, offsets, dw)) { std::printf("gemm_grouped_wgrad returned %d\n", err); return 1; }
    drv::Check chk;
    for (int t = 0; t < T; t++)
        for (int n = 0; n < N; n++) {
            float golden = 7.0f;                                 // rows outside every group keep what they held
            for (int e = 0; e < E; e++)
                if (t >= off[e] && t < off[e + 1]) {
                    golden = 0.0f;
                    for (int k = 0; k < K; k++) golden += x(k, t) * w(n, k, e);
                }
            chk.one(golden, y(n, t));
        }
    for (int e = 0; e < E; e++)
        for (int k = 0; k < K; k++)
            for (int n = 0; n < N; n++) {
                float golden = 0.0f;
                for (int t = off[e]; t < off[e + 1]; t++) golden += x(k, t) * dy(n, t);
                chk.one(golden, dw(n, k, e));
            }
    return chk.report("gemm_grouped", ns);
}
