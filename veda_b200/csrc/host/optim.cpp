// veda::optim on the device (src/libs/optim/AdamW.cpp, Clip.cpp).
#include "veda/optim.hpp"

#include "veda_cuda.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <unordered_set>

namespace veda::optim
{

using core::DType;
using core::Shape;
using core::Tensor;

namespace
{
cudaStream_t cs() { return reinterpret_cast<cudaStream_t>(current_stream()); }

float* fptr(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }

// The runs launch through device addresses taken once: bring any value or gradient the host wrote
// through Tensor::data() since then back to the device first (a no-op without host mirrors).
void flush_host_writes(const std::vector<autograd::Variable>& parameters)
{
    for (const auto& p : parameters)
    {
        p.value().storage()->data();
        if (p.node()->grad.defined())
        {
            p.node()->grad.storage()->data();
        }
    }
}
} // namespace

AdamW::AdamW(std::vector<autograd::Variable> parameters, AdamWConfig config)
    : parameters_(std::move(parameters)), config_(config)
{
    if (config_.learning_rate < 0.0f || config_.eps <= 0.0f || config_.weight_decay < 0.0f)
    {
        throw std::invalid_argument("AdamW: learning rate, eps and weight decay must be positive");
    }
    if (config_.beta1 < 0.0f || config_.beta1 >= 1.0f || config_.beta2 < 0.0f ||
        config_.beta2 >= 1.0f)
    {
        throw std::invalid_argument("AdamW: betas must lie in [0, 1)");
    }
    size_t total = 0, lowp_total = 0;
    for (const auto& p : parameters_)
    {
        total += p.value().numel();
        if (p.value().dtype() == DType::BF16)
        {
            lowp_total += p.value().numel();
        }
    }
    m_arena_ = Tensor(Shape({total > 0 ? total : 1}), DType::F32);
    v_arena_ = Tensor(Shape({total > 0 ? total : 1}), DType::F32);
    if (lowp_total > 0)
    {
        master_arena_ = Tensor::empty(Shape({lowp_total}), DType::F32);
    }
    size_t at = 0;
    for (const auto& p : parameters_)
    {
        if (p.value().dtype() == DType::BF16)
        {
            Tensor mview = Tensor::view(master_arena_.storage(), at, p.value().shape(), DType::F32);
            // the master starts at the parameter's (bf16) value, widened exactly
            std::vector<int64_t> shape(p.value().shape().dims().begin(), p.value().shape().dims().end());
            std::vector<int64_t> strides(p.value().strides().begin(), p.value().strides().end());
            if (shape.empty()) { shape = {1}; strides = {1}; }
            check(veda_copy_strided(p.value().storage()->data(), VEDA_BF16, strides.data(),
                                    static_cast<int64_t>(p.value().offset()), mview.data_ptr(),
                                    VEDA_F32, shape.data(), static_cast<int>(shape.size()),
                                    current_stream()),
                  "AdamW: master copy");
            masters_.push_back(mview);
            at += p.value().numel();
        }
        else
        {
            masters_.push_back(p.value());
        }
    }
    sumsq_ = Tensor(Shape({2}), DType::F32);   // 8 bytes: one double
    bias_ = Tensor(Shape({4 * (parameters_.size() + 1)}), DType::F32);
    build_runs();
}

AdamW::~AdamW() = default;

std::vector<AdamW::Run> AdamW::runs_of(bool all) const
{
    std::vector<Run> runs;
    size_t offset = 0;
    for (size_t i = 0; i < parameters_.size(); ++i)
    {
        const auto& p = parameters_[i];
        const size_t n = p.value().numel();
        if (!p.requires_grad() || n == 0 || (!all && taken_[i]))
        {
            offset += n;
            continue;
        }
        const Tensor& g = p.grad();   // allocates zeros for a leaf that has none yet
        if (g.dtype() != DType::F32 || !g.is_contiguous() || !p.value().is_contiguous())
        {
            throw std::invalid_argument("AdamW: parameters need contiguous values and fp32 gradients");
        }
        Run r{i, 1, static_cast<int64_t>(n), fptr(g), fptr(masters_[i]), fptr(m_arena_) + offset,
              fptr(v_arena_) + offset,
              p.value().dtype() == DType::BF16 ? p.value().data_ptr() : nullptr, starts_[i], 0};
        if (!runs.empty())
        {
            Run& last = runs.back();
            const bool adjacent = last.first + last.count == i && (all || last.start == r.start) &&
                                  last.grad + last.n == r.grad && last.master + last.n == r.master &&
                                  last.m + last.n == r.m &&
                                  ((last.lowp == nullptr && r.lowp == nullptr) ||
                                   (last.lowp != nullptr && r.lowp != nullptr &&
                                    static_cast<char*>(last.lowp) + last.n * 2 ==
                                        static_cast<char*>(r.lowp)));
            if (adjacent)
            {
                last.count += 1;
                last.n += r.n;
                offset += n;
                continue;
            }
        }
        runs.push_back(r);
        offset += n;
    }
    return runs;
}

void AdamW::build_runs()
{
    taken_.resize(parameters_.size(), false);
    starts_.resize(parameters_.size(), 0);
    runs_ = runs_of(true);
    build_updates();
    int64_t largest = 1;
    for (const Run& r : runs_)
    {
        largest = std::max<int64_t>(largest, r.n);
    }
    const size_t ws = veda_sumsq_workspace(largest);
    workspace_ = Tensor::empty(Shape({(ws + 3) / 4 + 1}), DType::F32);
}

void AdamW::set_taken(const std::vector<size_t>& indices, bool taken)
{
    for (const size_t i : indices)
    {
        taken_[i] = taken;
    }
    build_updates();
}

void AdamW::build_updates()
{
    std::vector<Run> updates = runs_of(false);
    std::vector<size_t> starts;
    for (Run& r : updates)
    {
        const auto at = std::find(starts.begin(), starts.end(), r.start);
        r.bias = static_cast<size_t>(at - starts.begin());
        if (at == starts.end())
        {
            starts.push_back(r.start);
        }
    }
    bias_host_.resize(2 * starts.size());
    updates_ = std::move(updates);
    bias_starts_ = std::move(starts);
    upload_bias();   // a step that is counted already finds its corrections in the new order
}

void AdamW::upload_bias()
{
    for (size_t k = 0; k < bias_starts_.size(); ++k)
    {
        // before the first step there is nothing to correct
        const double t = static_cast<double>(steps_ > bias_starts_[k] ? steps_ - bias_starts_[k] : 1);
        bias_host_[2 * k] = 1.0 - std::pow(static_cast<double>(config_.beta1), t);
        bias_host_[2 * k + 1] = 1.0 - std::pow(static_cast<double>(config_.beta2), t);
    }
    if (!bias_host_.empty() &&
        cudaMemcpyAsync(bias_.data_ptr(), bias_host_.data(), bias_host_.size() * sizeof(double), cudaMemcpyHostToDevice,
                        cs()) != cudaSuccess)
    {
        throw std::runtime_error("AdamW: bias correction upload failed");
    }
}

void AdamW::set_steps(size_t steps)
{
    steps_ = steps;
    bool changed = false;
    for (size_t& start : starts_)
    {
        changed = changed || start > steps;
        start = std::min(start, steps);
    }
    if (changed)
    {
        build_updates();
    }
}

void AdamW::set_starts(const std::vector<size_t>& starts)
{
    if (starts.size() != parameters_.size())
    {
        throw std::invalid_argument("AdamW::set_starts: " + std::to_string(starts.size()) + " starts for " +
                                    std::to_string(parameters_.size()) + " parameters");
    }
    starts_ = starts;
    build_updates();
}

void AdamW::restart(const std::vector<size_t>& indices)
{
    std::vector<size_t> starts = starts_;
    std::vector<size_t> offsets;
    size_t at = 0;
    for (const auto& p : parameters_)
    {
        offsets.push_back(at);
        at += p.value().numel();
    }
    for (const size_t i : indices)
    {
        const size_t bytes = parameters_.at(i).value().numel() * sizeof(float);
        if (bytes > 0 && (cudaMemsetAsync(fptr(m_arena_) + offsets[i], 0, bytes, cs()) != cudaSuccess ||
                          cudaMemsetAsync(fptr(v_arena_) + offsets[i], 0, bytes, cs()) != cudaSuccess))
        {
            throw std::runtime_error("AdamW::restart: memset failed");
        }
        starts[i] = steps_;
    }
    set_starts(starts);
}

void AdamW::advance()
{
    ++steps_;
    upload_bias();
}

void AdamW::launch(const double* sumsq, float max_norm, float grad_scale)
{
    flush_host_writes(parameters_);
    const double* bias = static_cast<const double*>(bias_.data_ptr());
    for (const Run& r : updates_)
    {
        check(veda_adamw_step_dev(r.master, r.m, r.v, r.grad, r.lowp, r.n, config_.learning_rate,
                                  config_.beta1, config_.beta2, config_.eps, config_.weight_decay,
                                  bias + 2 * r.bias, sumsq, max_norm, grad_scale,
                                  skip_nonfinite_ && sumsq != nullptr ? VEDA_ADAMW_SKIP_NONFINITE : 0,
                                  current_stream()),
              "AdamW::step");
    }
}

void AdamW::step()
{
    advance();
    launch(nullptr, 1.0f, 1.0f);
}

void AdamW::step_clipped(float max_norm, float grad_scale)
{
    advance();
    launch_clipped(max_norm, grad_scale);
}

void AdamW::launch_clipped(float max_norm, float grad_scale)
{
    if (!(max_norm > 0.0f))
    {
        throw std::invalid_argument("clip_gradient_norm: max_norm must be positive");
    }
    flush_host_writes(parameters_);
    double* ss = static_cast<double*>(sumsq_.data_ptr());
    for (size_t k = 0; k < runs_.size(); ++k)
    {
        check(veda_sumsq(runs_[k].grad, runs_[k].n, ss, k == 0 ? 0 : 1, workspace_.data_ptr(),
                         workspace_.numel() * 4, current_stream()),
              "AdamW::step_clipped (norm)");
    }
    last_scale_ = grad_scale;
    launch(ss, max_norm, grad_scale);
}

float AdamW::last_grad_norm()
{
    double ss = 0.0;
    if (cudaMemcpyAsync(&ss, sumsq_.data_ptr(), sizeof(double), cudaMemcpyDeviceToHost, cs()) !=
            cudaSuccess ||
        cudaStreamSynchronize(cs()) != cudaSuccess)
    {
        throw std::runtime_error("AdamW::last_grad_norm: read failed");
    }
    return static_cast<float>(std::sqrt(ss) * std::fabs(static_cast<double>(last_scale_)));
}

void AdamW::zero_grad()
{
    for (auto& p : parameters_)
    {
        if (!p.requires_grad())
        {
            continue;
        }
        auto& node = *p.node();
        if (node.grad.defined())
        {
            if (cudaMemsetAsync(node.grad.data_ptr(), 0, node.grad.numel() * 4, cs()) != cudaSuccess)
            {
                throw std::runtime_error("AdamW::zero_grad: memset failed");
            }
            node.grad_zero = true;
            node.grad_owned = true;
        }
    }
}

namespace
{
// Clears the gradients of the parameters that have one.
void clear_grads(const std::vector<autograd::Variable>& parameters, const char* what)
{
    for (const auto& p : parameters)
    {
        auto& node = *p.node();
        if (p.requires_grad() && node.grad.defined())
        {
            if (cudaMemsetAsync(node.grad.data_ptr(), 0, node.grad.numel() * 4, cs()) != cudaSuccess)
            {
                throw std::runtime_error(std::string(what) + ": memset failed");
            }
            node.grad_zero = true;
            node.grad_owned = true;
        }
    }
}

// A batch's scratch is about 8 bytes per weight; larger batches are cut so that it stays below this.
constexpr size_t kMuonWorkspace = size_t{1} << 30;
} // namespace

void Muon::check_config(const MuonConfig& c)
{
    if (!(c.learning_rate >= 0.0f) || !(c.weight_decay >= 0.0f) || !(c.eps >= 0.0f))
    {
        throw std::invalid_argument("Muon: learning rate, eps and weight decay must not be negative");
    }
    if (!(c.momentum >= 0.0f) || c.momentum >= 1.0f)
    {
        throw std::invalid_argument("Muon: momentum must lie in [0, 1)");
    }
    if (c.steps == 0 || c.steps > 64)   // veda_muon_step's range, refused before a step is half made
    {
        throw std::invalid_argument("Muon: 1 to 64 Newton-Schulz steps");
    }
}

void Muon::set_config(const MuonConfig& config)
{
    check_config(config);
    const bool other = config.fp32_products != config_.fp32_products;
    config_ = config;
    if (other)
    {
        build_batches();   // their workspace is another
    }
}

void Muon::check_parameters() const
{
    std::unordered_set<const void*> seen;
    for (const auto& p : parameters_)
    {
        if (!seen.insert(p.node().get()).second)
        {
            throw std::invalid_argument("Muon: a parameter is given twice");
        }
        if (p.value().rank() != 2)
        {
            throw std::invalid_argument("Muon: a parameter of shape " + p.value().shape().to_string() +
                                        " is not a matrix");
        }
    }
}

Muon::Muon(std::vector<autograd::Variable> parameters, MuonConfig config)
    : parameters_(std::move(parameters)), config_(config)
{
    check_config(config_);
    check_parameters();
    // Momentum and masters lie as the gradients do where those are views of one arena, so that equal
    // matrices at a constant distance stay so; back to back where the gradients are scattered.
    size_t total = 0;
    uintptr_t low = UINTPTR_MAX, high = 0;
    for (const auto& p : parameters_)
    {
        const uintptr_t at = reinterpret_cast<uintptr_t>(fptr(p.grad()));
        low = std::min(low, at);
        high = std::max(high, at + p.value().numel() * sizeof(float));
        total += p.value().numel();
    }
    const size_t span = total > 0 ? (high - low) / sizeof(float) : 0;
    const bool together = span <= total + total / 2 + 4096;
    const bool bf16 = !parameters_.empty() && parameters_[0].value().dtype() == DType::BF16;
    Tensor momentum(Shape({std::max<size_t>(1, together ? span : total)}), DType::F32);
    Tensor master;
    for (const auto& p : parameters_)
    {
        if ((p.value().dtype() == DType::BF16) != bf16)
        {
            throw std::invalid_argument("Muon: parameters of one dtype");
        }
    }
    if (bf16)
    {
        master = Tensor(Shape({std::max<size_t>(1, together ? span : total)}), DType::F32);
    }
    size_t at = 0;
    for (const auto& p : parameters_)
    {
        const size_t offset =
            together ? (reinterpret_cast<uintptr_t>(fptr(p.grad())) - low) / sizeof(float) : at;
        at += p.value().numel();
        momenta_.push_back(Tensor::view(momentum.storage(), offset, p.value().shape(), DType::F32));
        if (!bf16)
        {
            masters_.push_back(p.value());
            continue;
        }
        Tensor w = Tensor::view(master.storage(), offset, p.value().shape(), DType::F32);
        const int64_t shape[2] = {static_cast<int64_t>(p.value().shape()[0]),
                                  static_cast<int64_t>(p.value().shape()[1])};
        const int64_t strides[2] = {static_cast<int64_t>(p.value().strides()[0]),
                                    static_cast<int64_t>(p.value().strides()[1])};
        check(veda_copy_strided(p.value().storage()->data(), VEDA_BF16, strides,
                                static_cast<int64_t>(p.value().offset()), w.data_ptr(), VEDA_F32, shape, 2,
                                current_stream()),
              "Muon: master copy");
        masters_.push_back(w);
    }
    build_batches();
}

Muon::Muon(AdamW& base, const std::vector<size_t>& indices, MuonConfig config) : config_(config)
{
    size_t at = 0;
    std::vector<size_t> offsets;
    for (const auto& p : base.parameters())
    {
        offsets.push_back(at);
        at += p.value().numel();
    }
    for (const size_t i : indices)
    {
        if (i >= base.parameters().size())
        {
            throw std::invalid_argument("Muon: no parameter " + std::to_string(i));
        }
        if (base.taken_[i])
        {
            throw std::invalid_argument("Muon: parameter " + std::to_string(i) + " is taken already");
        }
        const auto& p = base.parameters()[i];
        parameters_.push_back(p);
        momenta_.push_back(Tensor::view(base.first_moments().storage(), offsets[i], p.value().shape(), DType::F32));
        masters_.push_back(base.master(i));
    }
    check_config(config_);
    check_parameters();
    build_batches();
    base.set_taken(indices, true);
    base_ = &base;
    taken_ = indices;
}

Muon::~Muon()
{
    if (base_ != nullptr)
    {
        try
        {
            base_->restart(taken_);
            base_->set_taken(taken_, false);
        }
        catch (...)
        {
            // a device that fails here fails the next call too; a destructor has no other way to say so
        }
    }
}

void Muon::build_batches()
{
    // Elements from a to b if their values, masters, momenta and gradients lie equally far apart.
    const auto distance = [&](size_t a, size_t b, int64_t* out) {
        const auto step = [&](const Tensor& x, const Tensor& y) {
            return (static_cast<const char*>(y.data_ptr()) - static_cast<const char*>(x.data_ptr())) /
                   static_cast<int64_t>(core::dtype_size(x.dtype()));
        };
        const int64_t d = step(parameters_[a].grad(), parameters_[b].grad());
        *out = d;
        return d >= static_cast<int64_t>(parameters_[a].value().numel()) &&
               step(parameters_[a].value(), parameters_[b].value()) == d &&
               step(masters_[a], masters_[b]) == d && step(momenta_[a], momenta_[b]) == d;
    };
    batches_.clear();
    workspace_bytes_ = 0;
    std::vector<bool> done(parameters_.size(), false);
    size_t largest = 1;
    for (size_t i = 0; i < parameters_.size(); ++i)
    {
        const auto& p = parameters_[i];
        if (done[i] || !p.requires_grad() || p.value().numel() == 0)
        {
            continue;
        }
        const Tensor& g = p.grad();
        if (g.dtype() != DType::F32 || !g.is_contiguous() || !p.value().is_contiguous())
        {
            throw std::invalid_argument("Muon: parameters need contiguous values and fp32 gradients");
        }
        const Shape& shape = p.value().shape();
        const int64_t rows = static_cast<int64_t>(shape[0]), cols = static_cast<int64_t>(shape[1]);
        const bool lowp = p.value().dtype() == DType::BF16;
        const int d = lowp && !config_.fp32_products ? VEDA_BF16 : VEDA_F32;
        Batch b{i, 1, rows, cols, 0, fptr(masters_[i]), fptr(momenta_[i]), fptr(g),
                lowp ? p.value().data_ptr() : nullptr};
        size_t last = i;
        for (size_t j = i + 1; j < parameters_.size(); ++j)
        {
            int64_t step = 0;
            if (done[j] || !parameters_[j].requires_grad() || parameters_[j].value().shape() != shape ||
                parameters_[j].value().dtype() != p.value().dtype() || !distance(last, j, &step) ||
                (b.count > 1 && step != b.stride) ||
                veda_muon_step_workspace(b.count + 1, rows, cols, d) > kMuonWorkspace)
            {
                continue;
            }
            b.stride = step;
            b.count += 1;
            done[j] = true;
            last = j;
        }
        workspace_bytes_ = std::max(workspace_bytes_, veda_muon_step_workspace(b.count, rows, cols, d));
        largest = std::max(largest, p.value().numel());
        batches_.push_back(b);
    }
    workspace_ = Tensor::empty(Shape({workspace_bytes_ / 4 + 1}), DType::F32);
    sumsq_ = Tensor(Shape({2}), DType::F32);   // 8 bytes: one double
    norm_workspace_ = Tensor::empty(Shape({veda_sumsq_workspace(static_cast<int64_t>(largest)) / 4 + 1}), DType::F32);
}

void Muon::launch(const double* sumsq, float max_norm, float grad_scale)
{
    flush_host_writes(parameters_);
    const MuonConfig& c = config_;
    const int flags = (base_ != nullptr && base_->skip_nonfinite() ? VEDA_ADAMW_SKIP_NONFINITE : 0) |
                      (c.fp32_products ? VEDA_MUON_FP32_PRODUCTS : 0);
    for (const Batch& b : batches_)
    {
        const float rows = static_cast<float>(b.rows), cols = static_cast<float>(b.cols);
        const float scale = c.match_adamw ? 0.2f * std::sqrt(std::max(rows, cols))
                                          : std::sqrt(std::max(1.0f, rows / cols));
        check(veda_muon_step(b.master, b.momentum, b.grad, b.lowp, b.count, b.rows, b.cols, b.stride,
                             c.learning_rate, c.momentum, c.nesterov ? 1 : 0, c.weight_decay, scale,
                             static_cast<int>(c.steps), c.a, c.b, c.c, c.eps, sumsq, max_norm, grad_scale, flags,
                             workspace_.data_ptr(), workspace_bytes_, current_stream()),
              "Muon::step");
    }
}

void Muon::step() { launch(nullptr, 1.0f, 1.0f); }

void Muon::step_clipped(float max_norm, float grad_scale)
{
    if (!(max_norm > 0.0f))
    {
        throw std::invalid_argument("clip_gradient_norm: max_norm must be positive");
    }
    flush_host_writes(parameters_);
    double* ss = static_cast<double*>(sumsq_.data_ptr());
    bool first = true;
    for (const auto& p : parameters_)
    {
        if (p.requires_grad())
        {
            check(veda_sumsq(fptr(p.grad()), static_cast<int64_t>(p.value().numel()), ss, first ? 0 : 1,
                             norm_workspace_.data_ptr(), norm_workspace_.numel() * 4, current_stream()),
                  "Muon::step_clipped (norm)");
            first = false;
        }
    }
    launch(ss, max_norm, grad_scale);
}

size_t Muon::elements() const noexcept
{
    size_t n = 0;
    for (const Batch& b : batches_) n += static_cast<size_t>(b.count * b.rows * b.cols);
    return n;
}

double Muon::flops() const noexcept
{
    double sum = 0.0;
    for (const Batch& b : batches_)
    {
        const double m = static_cast<double>(std::min(b.rows, b.cols)), n = static_cast<double>(std::max(b.rows, b.cols));
        sum += static_cast<double>(b.count * static_cast<int64_t>(config_.steps)) * (m * m * n + m * m * m + 2.0 * m * m * n);
    }
    return sum;
}

void Muon::zero_grad() { clear_grads(parameters_, "Muon::zero_grad"); }

float clip_gradient_norm(const std::vector<autograd::Variable>& parameters, float max_norm)
{
    if (!(max_norm > 0.0f))
    {
        throw std::invalid_argument("clip_gradient_norm: max_norm must be positive");
    }
    int64_t largest = 1;
    for (const auto& p : parameters)
    {
        largest = std::max<int64_t>(largest, static_cast<int64_t>(p.value().numel()));
    }
    const size_t ws = veda_sumsq_workspace(largest);
    Tensor work = Tensor::empty(Shape({(ws + 3) / 4 + 1}), DType::F32);
    Tensor sumsq(Shape({2}), DType::F32);
    double* ss = static_cast<double*>(sumsq.data_ptr());
    bool first = true;
    std::vector<Tensor> grads;
    for (const auto& p : parameters)
    {
        if (!p.requires_grad())
        {
            continue;
        }
        Tensor g = p.grad();
        if (g.dtype() != DType::F32 || !g.is_contiguous())
        {
            throw std::invalid_argument("clip_gradient_norm: gradients must be contiguous fp32");
        }
        check(veda_sumsq(fptr(g), static_cast<int64_t>(g.numel()), ss, first ? 0 : 1,
                         work.data_ptr(), work.numel() * 4, current_stream()),
              "clip_gradient_norm");
        first = false;
        grads.push_back(g);
    }
    double host = 0.0;
    if (cudaMemcpyAsync(&host, ss, sizeof(double), cudaMemcpyDeviceToHost, cs()) != cudaSuccess ||
        cudaStreamSynchronize(cs()) != cudaSuccess)
    {
        throw std::runtime_error("clip_gradient_norm: read failed");
    }
    const double total = std::sqrt(host);
    if (!std::isfinite(total) || total <= static_cast<double>(max_norm))
    {
        return static_cast<float>(total);   // reported, nothing written
    }
    for (const Tensor& g : grads)
    {
        check(veda_clip_apply(fptr(g), static_cast<int64_t>(g.numel()), ss, max_norm,
                              current_stream()),
              "clip_gradient_norm");
    }
    return static_cast<float>(total);
}

} // namespace veda::optim
