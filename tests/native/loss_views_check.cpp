// autograd::linear_cross_entropy on operands that are views (column slices, weights that begin inside a
// buffer) and on a weight that other nodes share, through the C++ API on a GPU. Prints "ok <name>" or
// "FAIL <name>: ..." per check.
#include "veda/autograd.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <exception>
#include <string>

using namespace veda;
using autograd::Variable;
using core::DType;
using core::Shape;
using core::Tensor;

namespace
{
int failures = 0;
void report(const std::string& name, bool ok, const std::string& why = "")
{
    std::printf("%s %s%s%s\n", ok ? "ok" : "FAIL", name.c_str(), ok ? "" : ": ", ok ? "" : why.c_str());
    failures += ok ? 0 : 1;
}
// a fixed sequence in [-1, 1)
std::vector<float> numbers(size_t n, uint32_t seed, float scale)
{
    std::vector<float> v(n);
    for (auto& x : v)
    {
        seed = seed * 1664525u + 1013904223u;
        x = scale * (static_cast<float>(seed >> 8) / 8388608.0f - 1.0f);
    }
    return v;
}
std::vector<int64_t> words(size_t rows, size_t V)
{
    std::vector<int64_t> t(rows);
    for (size_t i = 0; i < rows; ++i) t[i] = static_cast<int64_t>((i * 37) % V);
    return t;
}

struct Result
{
    std::vector<float> loss, dx, dw;
};
Result run(const Tensor& x, const Tensor& w, const std::vector<int64_t>& targets)
{
    Variable xv = Variable::leaf(x), wv = Variable::leaf(w);
    Variable loss = autograd::linear_cross_entropy(xv, wv, targets);
    loss.backward();
    return {loss.value().to_host(), xv.grad().to_host(), wv.grad().to_host()};
}

// The same numbers contiguous and as views give the same bits: the operands are laid out, or read in
// place, and then multiplied alike.
void views(const std::string& name, DType type, size_t rows, size_t V, size_t D)
{
    const std::vector<int64_t> targets = words(rows, V);
    const Tensor x = core::to_dtype(Tensor::from_host(numbers(rows * D, 1, 1.0f), Shape({rows, D})), type);
    const Tensor w = core::to_dtype(Tensor::from_host(numbers(V * D, 2, 0.2f), Shape({V, D})), type);
    const std::vector<float> xh = x.to_host(), wh = w.to_host();
    const Result want = run(x, w, targets);
    for (const size_t off : {size_t{0}, size_t{1}, size_t{4}})
    {
        // columns off .. off + D of a buffer whose pitch is a multiple of 8 elements
        const size_t pitch = D + 8;
        std::vector<float> wide(rows * pitch, 7.0f), late(V * D + off, 7.0f);
        for (size_t r = 0; r < rows; ++r) std::copy(xh.begin() + r * D, xh.begin() + (r + 1) * D, wide.begin() + r * pitch + off);
        std::copy(wh.begin(), wh.end(), late.begin() + off);
        const Tensor xs = core::to_dtype(Tensor::from_host(wide, Shape({rows, pitch})), type).slice(1, off, D);
        const Tensor buffer = core::to_dtype(Tensor::from_host(late, Shape({late.size()})), type);
        const Tensor ws = Tensor::view(buffer.storage(), off, Shape({V, D}), type);
        for (int which = 1; which < 4; ++which)
        {
            const std::string full = name + "_from_" + std::to_string(off) + (which & 1 ? "_x" : "") + (which & 2 ? "_w" : "");
            try
            {
                const Result got = run(which & 1 ? xs : x, which & 2 ? ws : w, targets);
                report(full, got.loss == want.loss && got.dx == want.dx && got.dw == want.dw);
            }
            catch (const std::exception& e)
            {
                report(full, false, e.what());
            }
        }
    }
}

// A weight that is no leaf and that another node shares: its gradient may be held in its own type by the time the
// loss head's comes.
void shared(const std::string& name, DType type, size_t rows, size_t V, size_t D)
{
    const std::vector<int64_t> targets = words(rows, V);
    const Tensor x = core::to_dtype(Tensor::from_host(numbers(rows * D, 3, 1.0f), Shape({rows, D})), type);
    const Tensor w = core::to_dtype(Tensor::from_host(numbers(V * D, 4, 0.2f), Shape({V, D})), type);
    const auto grad = [&](int which) {
        Variable leaf = Variable::leaf(w), xv = Variable::leaf(x, false);
        Variable weight = autograd::mul(leaf, 1.0f);
        const auto head = [&] { return autograd::linear_cross_entropy(xv, weight, targets); };
        const auto other = [&] { return autograd::cross_entropy(autograd::linear(xv, autograd::mul(weight, 0.5f)), targets); };
        Variable loss = which == 0   ? head()
                        : which == 1 ? other()
                        : which == 2 ? autograd::add(head(), other())
                                     : autograd::add(other(), head());
        loss.backward();
        return leaf.grad().to_host();
    };
    const std::vector<float> a = grad(0), b = grad(1);
    // in bf16 each part, their sum and what is handed to the leaf are rounded (2^-8 each, of at most |a| + |b|)
    // beside the parts' own roundings by themselves; fp32 the same with 2^-24
    const double step = type == DType::BF16 ? 1.0 / 256.0 : 1.0 / 16777216.0;
    for (int which = 2; which < 4; ++which)
    {
        const std::vector<float> both = grad(which);
        double worst = 0.0;
        for (size_t i = 0; i < both.size(); ++i)
        {
            const double size = std::fabs(static_cast<double>(a[i])) + std::fabs(static_cast<double>(b[i]));
            worst = std::max(worst, std::fabs(both[i] - (static_cast<double>(a[i]) + b[i])) / (6.0 * step * size + 1e-30));
        }
        report(name + "_" + std::to_string(which - 2), worst <= 1.0, std::to_string(worst));
    }
}
} // namespace

int main(int argc, char** argv)
{
    const std::string only = argc > 1 ? argv[1] : "";
    for (const DType type : {DType::BF16, DType::F32})
    {
        const std::string t = type == DType::BF16 ? "bf16" : "f32";
        // a few rows, a small problem, and the tensor cores
        if (only.empty() || only == "views")
        {
            views("views_few_" + t, type, 3, 700, 64);
            views("views_small_" + t, type, 40, 300, 64);
            views("views_tiled_" + t, type, 300, 5000, 64);
        }
        if (only.empty() || only == "shared")
        {
            shared("shared_few_" + t, type, 3, 700, 64);
            shared("shared_small_" + t, type, 40, 300, 64);
            shared("shared_tiled_" + t, type, 300, 5000, 64);
        }
    }
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
