// GPU test of graphs of gated feed-forward blocks on the C++ host interface (include/deep8/Deep8.h) in both types and with every activation,
// against the same graphs in double on the host: blocks behind one another, whose residual stream is read at two depths, and a
// variable that several nodes read.  Prints one line per test; exits non-zero on a failure.
#include <cuda_fp16.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

#include "../../include/deep8/Deep8.h"

using namespace Deep8;

static int g_failed = 0;

// ---- the graph in double: every operation stores its value and leaves a closure that adds to its inputs' gradients
struct Mat {
    size_t rows, cols;
    std::vector<double> v, g;
    Mat(size_t r, size_t c) : rows(r), cols(c), v(r * c, 0.0), g(r * c, 0.0) {}
};
struct Tape {
    std::vector<std::function<void()>> back;
    void run() {
        for (size_t i = back.size(); i-- > 0;) back[i]();
    }
};

static std::vector<bool> keptElements(const DropoutMask& m, size_t n) {
    std::vector<bool> keep(n, true);
    if (m.p == 0) return keep;
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
static void act(Activation which, double a, double& value, double& slope) {
    const double s = 1 / (1 + std::exp(-a)), pi = std::acos(-1.0), k = std::sqrt(2 / pi);
    switch (which) {
    case Activation::SiLu: value = a * s; slope = s + a * s * (1 - s); break;
    case Activation::Gelu: {
        const double cdf = 0.5 * std::erfc(-a / std::sqrt(2.0));
        value = a * cdf; slope = cdf + a * std::exp(-a * a / 2) / std::sqrt(2 * pi); break;
    }
    case Activation::GeluTanh: {
        const double t = std::tanh(k * (a + 0.044715 * a * a * a));
        value = 0.5 * a * (1 + t); slope = 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * k * (1 + 3 * 0.044715 * a * a); break;
    }
    case Activation::ReLu: value = a > 0 ? a : 0; slope = a > 0; break;
    default: value = s; slope = s * (1 - s);
    }
}
static Mat* product(Tape& t, Mat* x, Mat* w, size_t first = 0) {  // x * rows [first, first + x->cols) of w
    Mat* y = new Mat(x->rows, w->cols);
    for (size_t i = 0; i < x->rows; ++i)
        for (size_t k = 0; k < x->cols; ++k)
            for (size_t j = 0; j < w->cols; ++j) y->v[i * w->cols + j] += x->v[i * x->cols + k] * w->v[(first + k) * w->cols + j];
    t.back.push_back([=] {
        for (size_t i = 0; i < x->rows; ++i)
            for (size_t k = 0; k < x->cols; ++k)
                for (size_t j = 0; j < w->cols; ++j) {
                    const double d = y->g[i * w->cols + j];
                    x->g[i * x->cols + k] += d * w->v[(first + k) * w->cols + j];
                    w->g[(first + k) * w->cols + j] += d * x->v[i * x->cols + k];
                }
    });
    return y;
}
static Mat* gated(Tape& t, Mat* x, Mat* w, Activation which, const DropoutMask& m) {  // w: both projections, one below the other
    Mat *a = product(t, x, w, 0), *u = product(t, x, w, x->cols), *h = new Mat(a->rows, a->cols);
    auto keep = keptElements(m, h->v.size());
    for (size_t i = 0; i < h->v.size(); ++i) {
        double value, slope;
        act(which, a->v[i], value, slope);
        h->v[i] = keep[i] ? value * u->v[i] / (1 - m.p) : 0;
    }
    t.back.push_back([=] {
        for (size_t i = 0; i < h->v.size(); ++i) {
            double value, slope;
            act(which, a->v[i], value, slope);
            const double d = keep[i] ? h->g[i] / (1 - m.p) : 0;
            a->g[i] += d * u->v[i] * slope;
            u->g[i] += d * value;
        }
    });
    return h;
}
static Mat* drop(Tape& t, Mat* x, const DropoutMask& m, Mat* residual) {
    Mat* y = new Mat(x->rows, x->cols);
    auto keep = keptElements(m, y->v.size());
    for (size_t i = 0; i < y->v.size(); ++i) y->v[i] = residual->v[i] + (keep[i] ? x->v[i] / (1 - m.p) : 0);
    t.back.push_back([=] {
        for (size_t i = 0; i < y->v.size(); ++i) {
            residual->g[i] += y->g[i];
            if (keep[i]) x->g[i] += y->g[i] / (1 - m.p);
        }
    });
    return y;
}
static Mat* norm(Tape& t, Mat* x, Mat* gain, double eps) {
    Mat* y = new Mat(x->rows, x->cols);
    const size_t c = x->cols;
    std::vector<double> rstd(x->rows);
    for (size_t i = 0; i < x->rows; ++i) {
        double s = 0;
        for (size_t j = 0; j < c; ++j) s += x->v[i * c + j] * x->v[i * c + j];
        rstd[i] = 1 / std::sqrt(s / c + eps);
        for (size_t j = 0; j < c; ++j) y->v[i * c + j] = x->v[i * c + j] * rstd[i] * gain->v[j];
    }
    t.back.push_back([=] {
        for (size_t i = 0; i < x->rows; ++i) {
            double along = 0;
            for (size_t j = 0; j < c; ++j) along += y->g[i * c + j] * gain->v[j] * x->v[i * c + j] * rstd[i] / c;
            for (size_t j = 0; j < c; ++j) {
                const double n = x->v[i * c + j] * rstd[i];
                x->g[i * c + j] += rstd[i] * (y->g[i * c + j] * gain->v[j] - n * along);
                gain->g[j] += y->g[i * c + j] * n;
            }
        }
    });
    return y;
}

// ---- both sides together
static std::vector<char> encode(const std::vector<double>& v, DType type) {
    std::vector<char> out(v.size() * (type == DType::Float16 ? 2 : 4));
    for (size_t i = 0; i < v.size(); ++i) {
        if (type == DType::Float16) {
            const __half h = __float2half((float)v[i]);
            std::memcpy(&out[2 * i], &h, 2);
        } else {
            const float f = (float)v[i];
            std::memcpy(&out[4 * i], &f, 4);
        }
    }
    return out;
}
static std::vector<double> decode(const std::vector<char>& b, DType type) {
    std::vector<double> v(b.size() / (type == DType::Float16 ? 2 : 4));
    for (size_t i = 0; i < v.size(); ++i) {
        if (type == DType::Float16) {
            __half h;
            std::memcpy(&h, &b[2 * i], 2);
            v[i] = __half2float(h);
        } else {
            float f;
            std::memcpy(&f, &b[4 * i], 4);
            v[i] = f;
        }
    }
    return v;
}
struct Leaf {
    Mat* mat;
    Variable* variable;
    std::string name;
};
struct Graph {
    EagerExecutor executor{DeviceType::GPU};
    DType type;
    Tape tape;
    std::vector<Leaf> leaves;
    explicit Graph(DType t) : type(t) {}
    Leaf leaf(const char* name, size_t batch, std::vector<size_t> dims, double scale, double around = 0) {
        const size_t cols = dims.back(), rows = (dims.size() == 2 ? dims[0] : 1) * batch;
        Leaf l{new Mat(rows, cols), &parameter(&executor, batch, dims, true, type), name};
        for (auto& e : l.mat->v) e = around + (std::rand() / (double)RAND_MAX * 2 - 1) * scale;
        const auto bytes = encode(l.mat->v, type);
        l.mat->v = decode(bytes, type);
        l.variable->feed(bytes.data());
        leaves.push_back(l);
        return l;
    }
    // y against want, then every leaf's gradient: relative, in norm
    void check(Variable& y, Mat* want, int stored) {
        auto close = [&](const std::vector<double>& got, const std::vector<double>& ref, const std::string& what) {
            double off = 0, size = 0;
            for (size_t i = 0; i < got.size(); ++i) {
                off += (got[i] - ref[i]) * (got[i] - ref[i]);
                size += ref[i] * ref[i];
            }
            // `stored` tensors in a row, each off by half a step; fp32 products by 2^-19 of their terms, twice per tensor at most
            const double tol = type == DType::Float16 ? stored * std::ldexp(1.0, -11) : stored * std::ldexp(1.0, -18);
            if (!(std::sqrt(off) <= tol * std::sqrt(size))) {
                std::printf("  %s: %.3g of its size, allowed %.3g\n", what.c_str(), std::sqrt(off / size), tol);
                ++g_failed;
            }
        };
        std::vector<double> dy(want->v.size());
        for (auto& e : dy) e = std::rand() / (double)RAND_MAX * 2 - 1;
        const auto bytes = encode(dy, type);
        want->g = decode(bytes, type);
        std::vector<char> out(bytes.size());
        y.fetch(out.data());
        close(decode(out, type), want->v, "value");
        tape.run();
        for (int walk = 0; walk < 2; ++walk) {  // the second over the same nodes: the same gradients
            executor.backward(&y, bytes.data(), false);
            for (auto& l : leaves) {
                std::vector<char> g(encode(l.mat->g, type).size());
                l.variable->fetchGradient(g.data());
                close(decode(g, type), l.mat->g, "gradient of " + l.name + (walk ? ", second walk" : ""));
            }
        }
    }
};
static DropoutMask mask(double p, unsigned long long offset) {
    DropoutMask m;
    m.p = p;
    m.seed = 0x0123456789abcdefull;
    m.offset = offset;
    return m;
}

// `depth` blocks behind one another: the stream between two of them is read by the next block's norm and by the addition behind it, which lie
// at different distances from the end
static void stack(DType type, int depth, Activation which, bool fuse, bool touch) {
    Graph g(type);
    g.executor.setFusion(fuse);
    g.executor.setFirstTouch(touch);
    const size_t rows = 9, cols = 16, width = 24;
    Leaf x = g.leaf("x", 1, {rows, cols}, 2);
    Variable* y = x.variable;
    Mat* ry = x.mat;
    for (int b = 0; b < depth; ++b) {
        const std::string tag = std::to_string(b);
        Leaf gain = g.leaf(("gain" + tag).c_str(), 1, {cols}, 0.3, 1), w = g.leaf(("w" + tag).c_str(), 2, {cols, width}, 0.5), w2 = g.leaf(("w2" + tag).c_str(), 1, {width, cols}, 0.4);
        const DropoutMask in = mask(b ? 0.25 : 0, 2 * b), out = mask(0.125, (1ull << 33) + b);
        Variable& n = rmsNorm(*y, *gain.variable, 1e-5f);
        Variable& h = gatedProduct(n, *w.variable, which, in);
        y = &dropout(h * *w2.variable, out, *y);
        ry = drop(g.tape, product(g.tape, gated(g.tape, norm(g.tape, ry, gain.mat, 1e-5f), w.mat, which, in), w2.mat), out, ry);
    }
    g.check(*y, ry, 10 * depth);
}
// one normalised variable read by two gated products and a plain one: the second contribution to its gradient is added while a projection's
// own is written
static void shared(DType type, Activation which) {
    Graph g(type);
    const size_t rows = 7, cols = 16, width = 24;
    Leaf x = g.leaf("x", 1, {rows, cols}, 2), gain = g.leaf("gain", 1, {cols}, 0.3, 1), wa = g.leaf("wa", 2, {cols, width}, 0.5), wb = g.leaf("wb", 2, {cols, width}, 0.5),
         wc = g.leaf("wc", 1, {cols, width}, 0.5);
    const DropoutMask a = mask(0.25, 1), b = mask(0, 2), c = mask(0.125, 3), d = mask(0.5, 4);
    Variable& n = rmsNorm(*x.variable, *gain.variable, 1e-5f);
    Variable& ha = gatedProduct(n, *wa.variable, which, a);
    Variable& hb = gatedProduct(n, *wb.variable, which, b);
    Variable& inner = dropout(ha, c, hb);
    Variable& y = dropout(n * *wc.variable, d, inner);
    Mat* rn = norm(g.tape, x.mat, gain.mat, 1e-5f);
    Mat *ra = gated(g.tape, rn, wa.mat, which, a), *rb = gated(g.tape, rn, wb.mat, which, b);
    Mat* ri = drop(g.tape, ra, c, rb);
    g.check(y, drop(g.tape, product(g.tape, rn, wc.mat), d, ri), 12);
}

int main() {
    std::srand(4321);
    auto run = [](const std::string& name, const std::function<void()>& f) {
        const int before = g_failed;
        try {
            f();
        } catch (const std::exception& e) {
            std::printf("  EXCEPTION: %s\n", e.what());
            ++g_failed;
        }
        std::printf("[%s] %s\n", g_failed == before ? "  OK  " : "FAILED", name.c_str());
        std::fflush(stdout);
    };
    const char* names[] = {"silu", "gelu", "gelu_tanh", "relu", "sigmoid"};
    for (DType type : {DType::Float32, DType::Float16}) {
        const std::string t = type == DType::Float16 ? "fp16 " : "fp32 ";
        for (int a = 0; a < 5; ++a) {
            run(t + "one block, " + names[a], [=] { stack(type, 1, (Activation)a, true, true); });
            run(t + "one variable read by three products, " + names[a], [=] { shared(type, (Activation)a); });
        }
        run(t + "two blocks", [=] { stack(type, 2, Activation::SiLu, true, true); });
        run(t + "three blocks, node by node, gradients zero-filled", [=] { stack(type, 3, Activation::Gelu, false, false); });
    }
    std::printf("%d failed\n", g_failed);
    return g_failed ? 1 : 0;
}
