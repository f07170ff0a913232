// What optim::Muon takes over from an AdamW and gives back, through the C++ API on a GPU. Prints "ok <name>" or
// "FAIL <name>: ..." per check.
#include "veda/autograd.hpp"
#include "veda/optim.hpp"
#include "veda_cuda.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <memory>
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
constexpr size_t kRows = 24, kCols = 40, kN = kRows * kCols;
Tensor matrix(uint32_t seed, DType type)
{
    return core::to_dtype(Tensor::from_host(numbers(kN, seed, 0.1f), Shape({kRows, kCols})), type);
}
// leaves the numbers of `seed` as the gradient
void fill(Variable& p, uint32_t seed)
{
    p.zero_grad();
    const Tensor g = core::to_dtype(Tensor::from_host(numbers(kN, seed, 1.0f), Shape({kRows, kCols})), p.value().dtype());
    autograd::sum(autograd::mul(p, Variable::leaf(g, false))).backward();
}

void run(const std::string& name, DType type)
{
    const optim::AdamWConfig config{0.01f, 0.9f, 0.999f, 1e-8f, 0.1f};
    Variable a = Variable::leaf(matrix(1, type)), b = Variable::leaf(matrix(2, type)), c = Variable::leaf(matrix(3, type));
    Variable a2 = Variable::leaf(matrix(1, type)), c2 = Variable::leaf(matrix(3, type));
    optim::AdamW adam({a, b, c}, config), beside({a2, c2}, config);
    auto muon = std::make_unique<optim::Muon>(adam, std::vector<size_t>{1});
    uint32_t seed = 100;
    const auto all = [&](bool with_b) {
        ++seed;
        fill(a, seed);
        fill(a2, seed);
        if (with_b) fill(b, seed + 1000);
        fill(c, seed + 2000);
        fill(c2, seed + 2000);
    };
    for (int k = 0; k < 30; ++k)
    {
        all(true);
        adam.step();
        muon->launch(nullptr, 1.0f, 1.0f);
        beside.step();
    }
    // other numbers for the same parameters: the momentum stays
    const std::vector<float> momentum = muon->momentum(0).to_host();
    optim::MuonConfig other;
    other.learning_rate = 0.02f;
    muon->set_config(other);
    report(name + "_set_config_keeps_momentum", muon->momentum(0).to_host() == momentum && muon->config().learning_rate == 0.02f);
    other.momentum = 1.0f;
    bool refused = false;
    try
    {
        muon->set_config(other);
    }
    catch (const std::invalid_argument&)
    {
        refused = true;
    }
    report(name + "_set_config_refuses", refused && muon->config().momentum == 0.95f);
    muon.reset();
    // from here AdamW's steps on b are those of a new AdamW that starts with b's weights
    const std::vector<float> m0 = adam.first_moments().to_host(), v0 = adam.second_moments().to_host();
    bool clear = true;
    for (size_t i = kN; i < 2 * kN; ++i) clear = clear && m0[i] == 0.0f && v0[i] == 0.0f;
    report(name + "_moments_cleared", clear);
    Variable fresh = Variable::leaf(core::contiguous(b.value()));
    optim::AdamW anew({fresh}, config);
    if (type == DType::BF16)
    {
        // the same master weights
        const Tensor from = adam.master(1), to = anew.master(0);
        const int64_t shape[1] = {static_cast<int64_t>(kN)}, strides[1] = {1};
        check(veda_copy_strided(from.storage()->data(), VEDA_F32, strides, static_cast<int64_t>(from.offset()), to.data_ptr(),
                                VEDA_F32, shape, 1, current_stream()),
              "masters");
    }
    std::vector<float> before = adam.master(1).to_host();
    for (int k = 0; k < 12; ++k)
    {
        all(true);
        fill(fresh, seed + 1000);
        adam.step();
        beside.step();
        anew.step();
        if (k == 0)
        {
            const std::vector<float> after = adam.master(1).to_host();
            double worst = 0.0;
            // AdamW's first step moves every weight by lr, beside the decay; a few roundings
            for (size_t i = 0; i < kN; ++i)
            {
                worst = std::max(worst, std::fabs(static_cast<double>(after[i]) - before[i]) / (0.01 * (1.0 + 0.1 * std::fabs(before[i]))));
            }
            report(name + "_first_step_is_bounded", worst <= 1.0 + 1e-4, std::to_string(worst));
        }
    }
    report(name + "_goes_on_as_a_new_adamw",
           adam.master(1).to_host() == anew.master(0).to_host() && b.value().to_host() == fresh.value().to_host());
    report(name + "_others_are_not_touched",
           a.value().to_host() == a2.value().to_host() && c.value().to_host() == c2.value().to_host());
    // taken again, with a fresh momentum of its own, and given back a second time
    {
        optim::Muon again(adam, {1});
        all(true);
        adam.step();
        beside.step();
        again.step();
    }
    const std::vector<float> b1 = adam.master(1).to_host();
    all(true);
    adam.step();
    beside.step();
    const std::vector<float> b2 = adam.master(1).to_host();
    double moved = 0.0;
    for (size_t i = 0; i < kN; ++i) moved = std::max(moved, std::fabs(static_cast<double>(b2[i]) - b1[i]));
    report(name + "_given_back_twice", moved > 0.005 && moved < 0.0105, std::to_string(moved));
    report(name + "_others_are_still_not_touched",
           a.value().to_host() == a2.value().to_host() && c.value().to_host() == c2.value().to_host());
}

// A step count set back to before the hand-back counts from there.
void counted_back()
{
    const optim::AdamWConfig config{0.01f, 0.9f, 0.999f, 1e-8f, 0.1f};
    Variable a = Variable::leaf(matrix(5, DType::F32));
    optim::AdamW adam({a}, config);
    {
        optim::Muon muon(adam, {0});
        for (uint32_t k = 0; k < 5; ++k)
        {
            fill(a, 300 + k);
            adam.step();
            muon.step();
        }
    }
    report("starts_at_the_hand_back", adam.start(0) == 5 && !adam.taken(0));
    adam.set_steps(2);
    report("start_follows_the_count", adam.start(0) == 2 && adam.steps() == 2);
    Variable b = Variable::leaf(core::contiguous(a.value()));
    optim::AdamW anew({b}, config);
    for (uint32_t k = 0; k < 6; ++k)
    {
        fill(a, 400 + k);
        fill(b, 400 + k);
        adam.step();
        anew.step();
    }
    report("goes_on_from_the_count", a.value().to_host() == b.value().to_host());
}
} // namespace

int main()
{
    counted_back();
    run("f32", DType::F32);
    run("bf16", DType::BF16);
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
