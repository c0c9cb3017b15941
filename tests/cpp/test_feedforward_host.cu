// GPU test of the C++ host interface's nodes of a gated feed-forward block (include/deep8/Deep8.h: GatedProduct, Dropout, RMSNorm).
// Prints one line per test; exits non-zero on a failure.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <stdexcept>
#include <vector>

#include "../../include/deep8/Deep8.h"

using namespace Deep8;

static int g_failed = 0;
#define EXPECT(cond)                                                        \
    do {                                                                    \
        if (!(cond)) {                                                      \
            std::printf("  %s:%d: not true: %s\n", __FILE__, __LINE__, #cond); \
            ++g_failed;                                                     \
        }                                                                   \
    } while (0)
static bool same(const std::vector<float>& a, const std::vector<float>& b) { return a == b; }

// ---- the gated feed-forward block as a graph, y = r + dropout(gatedProduct(rmsNorm(r)) * w2), against plain loops in double: value and every
// gradient; the residual's gradient is the sum of two paths
static std::vector<bool> keptElements(const DropoutMask& m, size_t n) {
    std::vector<bool> keep(n);
    for (size_t i = 0; i < n; ++i) {  // Philox4x32-10
        unsigned c[4] = {(unsigned)(i / 4), (unsigned)((i / 4) >> 32), (unsigned)m.offset, (unsigned)(m.offset >> 32)};
        unsigned k0 = (unsigned)m.seed, k1 = (unsigned)(m.seed >> 32);
        for (int r = 0; r < 10; ++r, k0 += 0x9E3779B9u, k1 += 0xBB67AE85u) {
            unsigned long long a = 0xD2511F53ull * c[0], b = 0xCD9E8D57ull * c[2];
            unsigned n0 = (unsigned)(b >> 32) ^ c[1] ^ k0, n2 = (unsigned)(a >> 32) ^ c[3] ^ k1;
            c[0] = n0; c[1] = (unsigned)b; c[2] = n2; c[3] = (unsigned)a;
        }
        keep[i] = c[i % 4] >= m.p * 4294967296.0;
    }
    return keep;
}
static void gatedBlockGraph(bool fuse, bool touch) {
    EagerExecutor executor(DeviceType::GPU);
    executor.setFusion(fuse);
    executor.setFirstTouch(touch);
    const size_t rows = 7, cols = 12, width = 20;
    auto rnd = [](size_t n, double scale) {
        std::vector<float> v(n);
        for (auto& e : v) e = (float)((std::rand() / (double)RAND_MAX * 2 - 1) * scale);
        return v;
    };
    auto hr = rnd(rows * cols, 2), hg = rnd(cols, 1), hw = rnd(2 * cols * width, 0.5), hw2 = rnd(width * cols, 0.5), hdy = rnd(rows * cols, 1);
    Variable& r = parameter(&executor, {rows, cols});
    Variable& gain = parameter(&executor, {cols});
    Variable& w = parameter(&executor, 2, {cols, width});
    Variable& w2 = parameter(&executor, {width, cols});
    r.feed(hr.data()); gain.feed(hg.data()); w.feed(hw.data()); w2.feed(hw2.data());
    DropoutMask inner, outer;
    inner.p = 0.25; inner.seed = 99; inner.offset = 1;
    outer.p = 0.5; outer.seed = 99; outer.offset = 1ull << 40;
    Variable& n = rmsNorm(r, gain, 1e-5f);
    Variable& h = gatedProduct(n, w, Activation::SiLu, inner);
    Variable& z = h * w2;
    Variable& y = dropout(z, outer, r);
    std::vector<float> gy(rows * cols);
    y.fetch(gy.data());
    executor.backward(&y, hdy.data(), false);
    std::vector<float> gdr(rows * cols), gdg(cols), gdw(2 * cols * width), gdw2(width * cols);
    r.fetchGradient(gdr.data()); gain.fetchGradient(gdg.data()); w.fetchGradient(gdw.data()); w2.fetchGradient(gdw2.data());
    // the same in double
    auto kin = keptElements(inner, rows * width), kout = keptElements(outer, rows * cols);
    std::vector<double> rn(rows * cols), rstd(rows), a(rows * width), u(rows * width), rh(rows * width), ry(rows * cols), dz(rows * cols), dh(rows * width, 0.0);
    std::vector<double> dw(2 * cols * width, 0.0), dw2(width * cols, 0.0), dn(rows * cols, 0.0), dr(rows * cols), dg(cols, 0.0);
    for (size_t i = 0; i < rows; ++i) {
        double s = 0;
        for (size_t c = 0; c < cols; ++c) s += (double)hr[i * cols + c] * hr[i * cols + c];
        rstd[i] = 1 / std::sqrt(s / cols + 1e-5f);
        for (size_t c = 0; c < cols; ++c) rn[i * cols + c] = hr[i * cols + c] * rstd[i] * hg[c];
        for (size_t f = 0; f < width; ++f) {
            double pa = 0, pu = 0;
            for (size_t c = 0; c < cols; ++c) {
                pa += rn[i * cols + c] * hw[c * width + f];
                pu += rn[i * cols + c] * hw[(cols + c) * width + f];
            }
            a[i * width + f] = pa;
            u[i * width + f] = pu;
            rh[i * width + f] = kin[i * width + f] ? pa / (1 + std::exp(-pa)) * pu / 0.75 : 0;
        }
        for (size_t c = 0; c < cols; ++c) {
            double s2 = 0;
            for (size_t f = 0; f < width; ++f) s2 += rh[i * width + f] * hw2[f * cols + c];
            const size_t at = i * cols + c;
            ry[at] = hr[at] + (kout[at] ? s2 / 0.5 : 0);
            dz[at] = kout[at] ? hdy[at] / 0.5 : 0;
        }
        for (size_t f = 0; f < width; ++f) {
            for (size_t c = 0; c < cols; ++c) {
                dh[i * width + f] += dz[i * cols + c] * hw2[f * cols + c];
                dw2[f * cols + c] += rh[i * width + f] * dz[i * cols + c];
            }
            const double d = kin[i * width + f] ? dh[i * width + f] / 0.75 : 0, sg = 1 / (1 + std::exp(-a[i * width + f]));
            const double da = d * u[i * width + f] * (sg + a[i * width + f] * sg * (1 - sg)), du = d * a[i * width + f] * sg;
            for (size_t c = 0; c < cols; ++c) {
                dw[c * width + f] += rn[i * cols + c] * da;
                dw[(cols + c) * width + f] += rn[i * cols + c] * du;
                dn[i * cols + c] += da * hw[c * width + f] + du * hw[(cols + c) * width + f];
            }
        }
        double along = 0;
        for (size_t c = 0; c < cols; ++c) along += dn[i * cols + c] * hg[c] * hr[i * cols + c] * rstd[i] / cols;
        for (size_t c = 0; c < cols; ++c) {
            const double xn = hr[i * cols + c] * rstd[i];
            dr[i * cols + c] = hdy[i * cols + c] + rstd[i] * (dn[i * cols + c] * hg[c] - xn * along);
            dg[c] += dn[i * cols + c] * xn;
        }
    }
    // eight stored fp32 tensors in a row and sums of at most 40 terms: far below 1e-5 of the largest element
    auto close = [](const std::vector<float>& got, const std::vector<double>& want) {
        double worst = 0, most = 0;
        for (size_t i = 0; i < got.size(); ++i) {
            worst = std::max(worst, std::fabs(got[i] - want[i]));
            most = std::max(most, std::fabs(want[i]));
        }
        return worst <= 1e-5 * most;
    };
    EXPECT(close(gy, ry));
    EXPECT(close(gdr, dr));
    EXPECT(close(gdg, dg));
    EXPECT(close(gdw, dw));
    EXPECT(close(gdw2, dw2));
    // a second walk over the same nodes: the same gradients (nothing of the forward pass was used up)
    executor.backward(&y, hdy.data(), false);
    std::vector<float> again(2 * cols * width);
    w.fetchGradient(again.data());
    EXPECT(same(again, gdw));
    executor.clearInterimNodes();
    // refusals
    auto refused = [](std::function<void()> f) {
        try {
            f();
        } catch (const std::invalid_argument&) {
            return true;
        }
        return false;
    };
    EXPECT(refused([&] { gatedProduct(r, w2); }));                 // not a batch of two
    EXPECT(refused([&] { rmsNorm(r, w2); }));
    EXPECT(refused([&] { dropout(r, outer, w2); }));
    DropoutMask bad;
    bad.p = 1.5;
    EXPECT(refused([&] { dropout(r, bad); }));
    executor.clearInterimNodes();
}

int main() {
    std::srand(1234);
    struct Case {
        const char* name;
        std::function<void()> run;
    };
    std::vector<Case> cases = {
        {"gated feed-forward block with dropout and residual, value and gradients", [] { gatedBlockGraph(true, true); }},
        {"the same node by node, gradients zero-filled", [] { gatedBlockGraph(false, false); }},
    };
    for (auto& c : cases) {
        int before = g_failed;
        try {
            c.run();
        } catch (const std::exception& e) {
            std::printf("  EXCEPTION: %s\n", e.what());
            ++g_failed;
        }
        std::printf("[%s] %s\n", g_failed == before ? "  OK  " : "FAILED", c.name);
        std::fflush(stdout);
    }
    std::printf("%d failed\n", g_failed);
    return g_failed ? 1 : 0;
}
