// CPU test of the argument checks of the C++ gradients of the gated feed-forward block (include/deep8/Deep8.h: Math::GatedProductGrad,
// Math::RMSNormGrad): tensors without memory, so a call that passes the checks ends at the question for the GPU.
#include <cstdio>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/deep8/Deep8.h"

using namespace Deep8;

static Tensor bare(size_t batch, std::vector<size_t> dims, DType type, Device* device = nullptr) {
    TensorStorage none;
    none.device = device;
    return Tensor(none, 0, batch, dims, ElementType::from(type));
}

int main() {
    const DType f32 = DType::Float32, f16 = DType::Float16;
    Device* other = reinterpret_cast<Device*>(64);  // never looked into
    int failed = 0;
    // whether the call ends at its own checks (true) or gets past them
    auto refused = [](const std::function<void()>& call) {
        try {
            call();
        } catch (const std::invalid_argument& e) {
            return std::string(e.what()).find("must live on a GPU device") == std::string::npos;
        }
        return false;
    };
    auto expect = [&](const char* what, bool wanted, const std::function<void()>& call) {
        const bool ok = refused(call) == wanted;
        if (!ok) ++failed;
        std::printf("[%s] %s\n", ok ? "  OK  " : "FAILED", what);
    };

    Tensor x = bare(1, {4, 8}, f32), weight = bare(1, {8}, f32), dy = bare(1, {4, 8}, f32), dx = bare(1, {4, 8}, f32), dweight = bare(1, {8}, f32);
    Tensor halfDx = bare(1, {4, 8}, f16), halfDweight = bare(1, {8}, f16), halfDy = bare(1, {4, 8}, f16);
    Tensor farDx = bare(1, {4, 8}, f32, other), farDweight = bare(1, {8}, f32, other), farDy = bare(1, {4, 8}, f32, other);
    auto norm = [&](Tensor& a, Tensor& b, const Tensor& d) { return [&a, &b, &d, &x, &weight] { Math::RMSNormGrad(x, &a, weight, &b, nullptr, d, false, true); }; };
    expect("norm: matching tensors", false, norm(dx, dweight, dy));
    expect("norm: dx of another type", true, norm(halfDx, dweight, dy));
    expect("norm: dweight of another type", true, norm(dx, halfDweight, dy));
    expect("norm: dy of another type", true, norm(dx, dweight, halfDy));
    expect("norm: dx on another device", true, norm(farDx, dweight, dy));
    expect("norm: dweight on another device", true, norm(dx, farDweight, dy));
    expect("norm: dy on another device", true, norm(dx, dweight, farDy));
    expect("norm: dx of another shape", true, norm(dweight, dweight, dy));

    Tensor w = bare(2, {8, 6}, f32), dw = bare(2, {8, 6}, f32), dz = bare(1, {4, 6}, f32), farDw = bare(2, {8, 6}, f32, other), halfDw = bare(2, {8, 6}, f16);
    auto gated = [&](Tensor& a, Tensor& b) {
        return [&a, &b, &x, &w, &dz] { Math::GatedProductGrad(x, &a, w, &b, Activation::SiLu, DropoutMask(), nullptr, nullptr, dz, false, true); };
    };
    expect("gated: matching tensors", false, gated(dx, dw));
    expect("gated: dx of another type", true, gated(halfDx, dw));
    expect("gated: dw of another type", true, gated(dx, halfDw));
    expect("gated: dx on another device", true, gated(farDx, dw));
    expect("gated: dw on another device", true, gated(dx, farDw));
    std::printf("%d failed\n", failed);
    return failed ? 1 : 0;
}
