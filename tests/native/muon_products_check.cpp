// optim::MuonConfig::fp32_products on bf16 parameters, through the C++ API on a GPU. Prints "ok <name>" or
// "FAIL <name>: ..." per check.
#include "veda/autograd.hpp"
#include "veda/optim.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>
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
} // namespace

int main()
{
    // the same steps with bf16 and with fp32 parameters that begin at the same values, on the same gradients
    const size_t rows = 300, cols = 264, n = rows * cols;
    const auto steps = [&](DType type, int fp32_from) {
        Tensor w = core::to_dtype(Tensor::from_host(numbers(n, 1, 0.1f), Shape({rows, cols})), DType::BF16);
        Variable p = Variable::leaf(core::to_dtype(w, type));
        optim::MuonConfig c;
        c.learning_rate = 0.01f;
        c.fp32_products = fp32_from == 0;
        optim::Muon muon({p}, c);
        for (int k = 0; k < 3; ++k)
        {
            if (k == fp32_from && k > 0)
            {
                c.fp32_products = true;
                muon.set_config(c);
            }
            p.zero_grad();
            const Tensor g = core::to_dtype(core::to_dtype(Tensor::from_host(numbers(n, 10 + k, 1.0f), Shape({rows, cols})), DType::BF16), type);
            autograd::sum(autograd::mul(p, Variable::leaf(g, false))).backward();
            muon.step();
        }
        return muon.master(0).to_host();
    };
    const std::vector<float> want = steps(DType::F32, 3), exact = steps(DType::BF16, 0), half = steps(DType::BF16, 3), mixed = steps(DType::BF16, 1);
    report("fp32_products_are_those_of_fp32_parameters", exact == want);
    const auto off = [&](const std::vector<float>& a) {
        double e = 0.0, s = 0.0;
        for (size_t i = 0; i < n; ++i)
        {
            e += std::pow(static_cast<double>(a[i]) - want[i], 2);
            s += std::pow(static_cast<double>(want[i]), 2);
        }
        return std::sqrt(e / s);
    };
    report("without_they_are_others", off(half) > 0.0 && off(half) < 1e-2, std::to_string(off(half)));
    report("set_config_switches", off(mixed) > 0.0 && off(mixed) < off(half), std::to_string(off(mixed)));
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
