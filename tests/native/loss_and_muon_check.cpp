// autograd::linear_cross_entropy against cross_entropy(linear(..)) and central differences, and
// optim::Muon on its own and beside AdamW, through the C++ API on a GPU. Prints "ok <name>" or
// "FAIL <name>: ..." per check.
#include "veda/autograd.hpp"
#include "veda/optim.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <functional>
#include <stdexcept>
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
double worst(const std::vector<float>& a, const std::vector<float>& b)
{
    double top = 0.0, off = 0.0;
    for (size_t i = 0; i < a.size(); ++i)
    {
        top = std::max(top, std::fabs(static_cast<double>(b[i])));
        off = std::max(off, std::fabs(static_cast<double>(a[i]) - b[i]));
    }
    return off / std::max(top, 1e-30);
}
template <typename E>
bool throws(const std::function<void()>& f)
{
    try
    {
        f();
    }
    catch (const E&)
    {
        return true;
    }
    catch (...)
    {
    }
    return false;
}
} // namespace

int main()
{
    const size_t rows = 12, V = 40, D = 24;
    const std::vector<float> xh = numbers(rows * D, 1, 1.0f), wh = numbers(V * D, 2, 0.5f);
    std::vector<int64_t> targets(rows);
    for (size_t i = 0; i < rows; ++i) targets[i] = static_cast<int64_t>((i * 7) % V);

    {
        // the same loss and gradients as the two nodes, in a graph that scales the loss and shares w
        auto run = [&](bool fused) {
            Variable x = Variable::leaf(Tensor::from_host(xh, Shape({3, 4, D})));
            Variable w = Variable::leaf(Tensor::from_host(wh, Shape({V, D})));
            Variable loss = fused ? autograd::linear_cross_entropy(x, w, targets)
                                  : autograd::cross_entropy(autograd::linear(x, w), targets);
            Variable total = autograd::add(autograd::mul(loss, -3.0f), autograd::mul(autograd::sum(w), 0.25f));
            total.backward();
            total.backward();   // leaf gradients accumulate across passes
            return std::vector<std::vector<float>>{loss.value().to_host(), x.grad().to_host(), w.grad().to_host()};
        };
        const auto a = run(true), b = run(false);
        // both in fp32: sums of 24, 40 and 12 terms; 64 steps of 2^-24 of the largest element
        const double tol = 64.0 / 16777216.0;
        for (size_t i = 0; i < a.size(); ++i)
        {
            report("fused_equals_composition_" + std::to_string(i), worst(a[i], b[i]) <= tol, std::to_string(worst(a[i], b[i])));
        }
    }
    {
        // ignored rows: the mean and the gradients of the others alone
        std::vector<int64_t> some = targets, few;
        std::vector<float> kept;
        for (size_t i = 0; i < rows; ++i)
        {
            if (i % 3 == 1)
            {
                some[i] = autograd::kIgnoreTarget;
                continue;
            }
            few.push_back(targets[i]);
            kept.insert(kept.end(), xh.begin() + i * D, xh.begin() + (i + 1) * D);
        }
        Variable x = Variable::leaf(Tensor::from_host(xh, Shape({rows, D})));
        Variable w = Variable::leaf(Tensor::from_host(wh, Shape({V, D})));
        Variable la = autograd::linear_cross_entropy(x, w, some);
        la.backward();
        Variable x2 = Variable::leaf(Tensor::from_host(kept, Shape({few.size(), D})));
        Variable w2 = Variable::leaf(Tensor::from_host(wh, Shape({V, D})));
        Variable lb = autograd::linear_cross_entropy(x2, w2, few);
        lb.backward();
        report("ignored_rows_loss", la.value().to_host() == lb.value().to_host());
        report("ignored_rows_weight_gradient", worst(w.grad().to_host(), w2.grad().to_host()) <= 64.0 / 16777216.0);
        const std::vector<float> gx = x.grad().to_host();
        bool zero = true;
        for (size_t i = 1; i < rows; i += 3)
        {
            for (size_t c = 0; c < D; ++c) zero = zero && gx[i * D + c] == 0.0f;
        }
        report("ignored_rows_input_gradient", zero);
    }
    {
        // Central differences against the tape, for x and for w. A loss between 2 and 4 is stored to half
        // a step of 2^-22 / 2 = 2^-23, and its rows carry some 4 roundings of 2^-24 x 4 (log-sum-exp,
        // target, difference): 1.1e-6 in all, over 2 h = 0.02 twice, so a difference is off by up to
        // 1.1e-4, 0.11 of the check's smallest scale of 1e-3.
        const float h = 1e-2f;
        const double tolerance = 0.11;
        const Tensor wt = Tensor::from_host(wh, Shape({V, D})), xt = Tensor::from_host(xh, Shape({rows, D}));
        const auto cx = autograd::check_gradient(
            [&](const Variable& x) { return autograd::linear_cross_entropy(x, Variable::leaf(wt, false), targets); }, xt, h,
            tolerance);
        report("differences_input", cx.ok, cx.message);
        const auto cw = autograd::check_gradient(
            [&](const Variable& w) { return autograd::linear_cross_entropy(Variable::leaf(xt, false), w, targets); }, wt, h,
            tolerance);
        report("differences_weight", cw.ok, cw.message);
    }
    {
        Variable x = Variable::leaf(Tensor::from_host(xh, Shape({rows, D})));
        Variable w = Variable::leaf(Tensor::from_host(wh, Shape({V, D})));
        std::vector<int64_t> outside = targets;
        outside[3] = static_cast<int64_t>(V);
        report("refuses_target", throws<std::invalid_argument>([&] { autograd::linear_cross_entropy(x, w, outside); }));
        report("refuses_count", throws<std::invalid_argument>([&] { autograd::linear_cross_entropy(x, w, {1, 2}); }));
        Variable narrow = Variable::leaf(Tensor::from_host(numbers(V * (D - 1), 3, 1.0f), Shape({V, D - 1})));
        report("refuses_width", throws<std::invalid_argument>([&] { autograd::linear_cross_entropy(x, narrow, targets); }));
        std::vector<float> packed(2 * rows);
        std::vector<int64_t> bad = targets;
        bad[5] = -7;
        std::copy(reinterpret_cast<const float*>(bad.data()), reinterpret_cast<const float*>(bad.data()) + 2 * rows,
                  packed.begin());
        const Tensor device = Tensor::from_host(packed, Shape({2 * rows}));
        Variable loss = autograd::linear_cross_entropy_device(x, w, device);
        report("flags_device_target", throws<std::out_of_range>([] { autograd::detail::raise_device_flag(); }));
    }
    {
        // Muon: three matrices of two shapes; one step moves each by lr weight_decay w + lr scale O with
        // O's singular values near 1, so |O|_F^2 lies between 0.45 and 1.3 times its rank
        std::vector<Variable> ps;
        std::vector<std::vector<float>> before;
        const size_t shapes[3][2] = {{20, 32}, {20, 32}, {48, 16}};
        for (uint32_t i = 0; i < 3; ++i)
        {
            const size_t n = shapes[i][0] * shapes[i][1];
            before.push_back(numbers(n, 10 + i, 0.1f));
            Variable p = Variable::leaf(Tensor::from_host(before.back(), Shape({shapes[i][0], shapes[i][1]})));
            autograd::sum(autograd::mul(p, Variable::leaf(Tensor::from_host(numbers(n, 20 + i, 1.0f), p.value().shape()), false))).backward();
            ps.push_back(p);
        }
        optim::MuonConfig c;
        c.learning_rate = 0.01f;
        c.weight_decay = 0.0f;
        c.match_adamw = false;
        optim::Muon muon(ps, c);
        muon.step();
        for (size_t i = 0; i < 3; ++i)
        {
            const std::vector<float> after = ps[i].value().to_host();
            const double scale = std::sqrt(std::max(1.0, static_cast<double>(shapes[i][0]) / shapes[i][1]));
            double sum = 0.0;
            for (size_t k = 0; k < after.size(); ++k)
            {
                const double o = (before[i][k] - after[k]) / (0.01 * scale);
                sum += o * o;
            }
            const double rank = static_cast<double>(std::min(shapes[i][0], shapes[i][1]));
            report("muon_moves_orthogonally_" + std::to_string(i), sum > 0.45 * rank && sum < 1.3 * rank, std::to_string(sum / rank));
            report("muon_momentum_" + std::to_string(i), muon.momentum(i).to_host() == ps[i].grad().to_host());
        }
        muon.zero_grad();
        report("muon_zero_grad", worst(ps[0].grad().to_host(), std::vector<float>(640, 0.0f)) == 0.0);
        Variable flat = Variable::leaf(Tensor::from_host(numbers(8, 1, 1.0f), Shape({8})));
        report("muon_refuses_vector", throws<std::invalid_argument>([&] { optim::Muon m({flat}); }));
        optim::MuonConfig bad;
        bad.momentum = 1.0f;
        report("muon_refuses_momentum", throws<std::invalid_argument>([&] { optim::Muon m(ps, bad); }));
        bad = {};
        bad.steps = 0;
        report("muon_refuses_no_steps", throws<std::invalid_argument>([&] { optim::Muon m(ps, bad); }));
        bad.steps = 65;
        report("muon_refuses_too_many_steps", throws<std::invalid_argument>([&] { optim::Muon m(ps, bad); }));
        report("muon_refuses_a_parameter_twice", throws<std::invalid_argument>([&] { optim::Muon m({ps[0], ps[0]}); }));
    }
    {
        // beside AdamW: a taken parameter is left to Muon, and given back with it
        auto fill = [](Variable& p, float v) {
            p.zero_grad();
            autograd::sum(autograd::mul(p, v)).backward();
        };
        Variable a = Variable::leaf(Tensor::from_host(numbers(64, 1, 0.1f), Shape({8, 8})));
        Variable b = Variable::leaf(Tensor::from_host(numbers(64, 2, 0.1f), Shape({8, 8})));
        optim::AdamW adam({a, b}, {0.01f, 0.9f, 0.999f, 1e-8f, 0.0f});
        const std::vector<float> b0 = b.value().to_host();
        {
            optim::Muon muon(adam, {1});
            fill(a, 1.0f);
            fill(b, 1.0f);
            adam.step_clipped(100.0f);
            report("taken_is_left_alone", b.value().to_host() == b0);
            report("norm_counts_taken", std::fabs(adam.last_grad_norm() - std::sqrt(128.0f)) < 1e-4f);
            muon.launch(adam.sumsq(), 100.0f, 1.0f);
            report("muon_updates_taken", b.value().to_host() != b0);
            report("refuses_taken_twice", throws<std::invalid_argument>([&] { optim::Muon again(adam, {1}); }));
            report("refuses_an_index_twice", throws<std::invalid_argument>([&] { optim::Muon again(adam, {0, 0}); }));
            report("refuses_index", throws<std::invalid_argument>([&] { optim::Muon again(adam, {2}); }));
        }
        const std::vector<float> b1 = b.value().to_host();
        adam.step();
        report("given_back", b.value().to_host() != b1);
    }
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
