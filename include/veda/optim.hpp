// veda::optim — AdamW and global-norm clipping with the reference's API and arithmetic
// (src/libs/optim/AdamW.h:23-59, AdamW.cpp:15-109; Clip.h:34, Clip.cpp:12-61) on device
// gradients.
//
// AdamW keeps fp32 first and second moments in two flat arenas and, for bf16 parameters, an fp32
// master copy (the parameter's bf16 value is rewritten from it after every step). Parameters
// whose gradients, values and masters lie back to back in memory — every parameter of
// train::TinyTransformer does — are updated by one kernel launch. step_clipped() fuses the
// global-norm clip into the update (the norm is computed on the device and read by the update
// kernel, no host round trip).
#pragma once

#include "veda/autograd.hpp"

#include <vector>

namespace veda::optim
{

struct AdamWConfig
{
    float learning_rate = 1e-3f;
    float beta1 = 0.9f;
    float beta2 = 0.999f;
    float eps = 1e-8f;
    float weight_decay = 0.01f;
};

class AdamW
{
public:
    explicit AdamW(std::vector<autograd::Variable> parameters, AdamWConfig config = {});
    ~AdamW();
    AdamW(const AdamW&) = delete;
    AdamW& operator=(const AdamW&) = delete;

    // The reference step: m, v, bias correction in double, decoupled decay first. Does not clear
    // the gradients.
    void step();
    // Clip to max_norm (the global norm of grad_scale * g) and step, in two launches per run of
    // contiguous parameters; nothing is synchronised. grad_scale carries a data-parallel 1/world.
    void step_clipped(float max_norm, float grad_scale = 1.0f);
    // step_clipped split in two for a step replayed from a CUDA graph: advance() counts the step
    // and leaves its bias corrections in device memory (not capturable: call it before each
    // replay); launch_clipped() only launches kernels, which read them there.
    void advance();
    void launch_clipped(float max_norm, float grad_scale = 1.0f);
    // The pre-clip global norm of the last step_clipped() (synchronises the stream).
    float last_grad_norm();
    void zero_grad();

    size_t steps() const noexcept { return steps_; }
    const AdamWConfig& config() const noexcept { return config_; }
    // First and second moments of every parameter, fp32, back to back in parameter order.
    const core::Tensor& first_moments() const noexcept { return m_arena_; }
    const core::Tensor& second_moments() const noexcept { return v_arena_; }
    // Restores the step count (the bias corrections of the next step use steps + 1, or what has been made since a
    // restart(), which lies no later than the count).
    void set_steps(size_t steps);
    // Steps that had been made when the moments of parameter i began: its bias corrections count from
    // there. 0 but for parameters that restart() was called for.
    size_t start(size_t i) const { return starts_.at(i); }
    void set_starts(const std::vector<size_t>& starts);
    // Clears the moments of these parameters; their bias corrections begin anew, as a new AdamW's do.
    void restart(const std::vector<size_t>& indices);
    // Whether a Muon has parameter i.
    bool taken(size_t i) const { return taken_.at(i); }
    // On: a clipped step whose global norm is not finite updates nothing (weights, moments and
    // gradients are left as they were); the caller, who reads the norm, then takes the step back
    // with set_steps(steps() - 1). Off (the default, the reference's behaviour): the step runs.
    void set_skip_nonfinite(bool on) noexcept { skip_nonfinite_ = on; }
    bool skip_nonfinite() const noexcept { return skip_nonfinite_; }
    const std::vector<autograd::Variable>& parameters() const noexcept { return parameters_; }
    // fp32 master weights of parameter i (the value itself for fp32 parameters).
    core::Tensor master(size_t i) const { return masters_[i]; }
    // Number of kernel launches one step issues (one per contiguous run).
    size_t runs() const noexcept { return updates_.size(); }
    // The device sum of squares that the last launch_clipped left (before grad_scale).
    const double* sumsq() const { return static_cast<const double*>(sumsq_.data_ptr()); }

private:
    bool skip_nonfinite_ = false;
    struct Run
    {
        size_t first, count;
        int64_t n;
        float* grad;
        float* master;
        float* m;
        float* v;
        void* lowp;   // bf16 value copy, or null for fp32 parameters
        size_t start, bias;   // steps before its moments began; its pair in bias_
    };
    friend class Muon;
    void build_runs();
    std::vector<Run> runs_of(bool all) const;
    // Leaves parameters to another optimizer, or takes them back.
    void set_taken(const std::vector<size_t>& indices, bool taken);
    void build_updates();
    void upload_bias();
    void launch(const double* sumsq, float max_norm, float grad_scale);

    std::vector<autograd::Variable> parameters_;
    std::vector<core::Tensor> masters_;
    core::Tensor m_arena_, v_arena_, master_arena_;
    std::vector<Run> runs_;      // every parameter: what the global norm covers
    std::vector<Run> updates_;   // those that step() updates
    std::vector<bool> taken_;
    std::vector<size_t> starts_;
    AdamWConfig config_;
    size_t steps_ = 0;
    core::Tensor sumsq_;     // device double
    // device doubles: 1 - beta1^t, 1 - beta2^t of the current step, a pair for each start in use (room for a
    // pair a parameter, so that the address stays)
    core::Tensor bias_;
    std::vector<size_t> bias_starts_;
    std::vector<double> bias_host_;
    core::Tensor workspace_;
    float last_scale_ = 1.0f;
};

struct MuonConfig
{
    float learning_rate = 3e-4f;
    float momentum = 0.95f;
    bool nesterov = true;
    float weight_decay = 0.1f;
    size_t steps = 5;              // Newton-Schulz iterations
    float a = 3.4445f, b = -4.7750f, c = 2.0315f;
    float eps = 1e-7f;
    // The orthogonalised update is scaled by 0.2 sqrt(max(rows, cols)), which gives its entries the
    // size of AdamW's, so learning rates carry over (false: by sqrt(max(1, rows / cols))).
    bool match_adamw = true;
    // bf16 parameters with both sides above 64: products as for fp32 ones (VEDA_MUON_FP32_PRODUCTS), which keeps the
    // master weights exact to fp32 at three times the operations; without, the update is off by some 0.15 %.
    bool fp32_products = false;
};

// Momentum orthogonalised by Newton-Schulz products (veda_muon_step) for rank-2 parameters:
//   m <- momentum m + g;  u = nesterov ? g + momentum m : m;
//   w <- w - lr weight_decay w - lr scale orthogonalize(u).
// Momentum and, for bf16 parameters, master weights are fp32. Parameters of one shape that lie a
// constant distance apart are updated as one batch: from each on, the next of its shape sets the distance and those
// that follow at it join. In train::TinyTransformer that makes one batch of a matrix that is the only one of its shape
// in a layer (down of every layer), and a pair a layer of two neighbours of one shape (k and v, gate and up).
// Not part of the reference, whose optimizer is AdamW. The method and the quintic's coefficients: K. Jordan et al.,
// "Muon: An optimizer for hidden layers in neural networks" (2024); the scale 0.2 sqrt(max(rows, cols)): J. Liu et
// al., "Muon is Scalable for LLM Training" (2025).
class Muon
{
public:
    // Keeps momentum and master weights of its own.
    explicit Muon(std::vector<autograd::Variable> parameters, MuonConfig config = {});
    // Takes over the parameters `indices` of an AdamW: its steps no longer update them (its global
    // norm still counts them), their momentum is their first moment there and their master weights
    // are its. `base` must outlive this object, whose end gives them back: the momentum, some 1 / (1 - momentum)
    // gradients in size and without a second moment beside it, is of no use to AdamW, so its moments for
    // them are cleared and their bias corrections begin anew (AdamW::restart).
    Muon(AdamW& base, const std::vector<size_t>& indices, MuonConfig config = {});
    ~Muon();
    Muon(const Muon&) = delete;
    Muon& operator=(const Muon&) = delete;

    // One step on the gradients as they are; does not clear them.
    void step();
    // The global-norm clip over these parameters fused into the step, as AdamW::step_clipped.
    void step_clipped(float max_norm, float grad_scale = 1.0f);
    // Only launches kernels (capturable): the step with the clip of a sum of squares in device memory
    // (null: none).
    void launch(const double* sumsq, float max_norm, float grad_scale);
    void zero_grad();
    const MuonConfig& config() const noexcept { return config_; }
    // Other numbers from the next launch on; momentum and master weights stay. A refused one changes nothing.
    void set_config(const MuonConfig& config);
    const std::vector<autograd::Variable>& parameters() const noexcept { return parameters_; }
    // fp32 momentum and master weights of parameter i (the value itself for fp32 parameters).
    core::Tensor momentum(size_t i) const { return momenta_[i]; }
    core::Tensor master(size_t i) const { return masters_[i]; }
    // Batches a step launches.
    size_t batches() const noexcept { return batches_.size(); }
    // Weights that a step updates, and the operations of its products (symmetric ones counted by halves).
    size_t elements() const noexcept;
    double flops() const noexcept;

private:
    struct Batch
    {
        size_t first;
        int64_t count, rows, cols, stride;
        float* master;
        float* momentum;
        float* grad;
        void* lowp;
    };
    static void check_config(const MuonConfig& config);
    void check_parameters() const;
    void build_batches();

    AdamW* base_ = nullptr;
    std::vector<size_t> taken_;
    std::vector<autograd::Variable> parameters_;
    std::vector<core::Tensor> momenta_, masters_;
    std::vector<Batch> batches_;
    MuonConfig config_;
    core::Tensor workspace_, sumsq_, norm_workspace_;
    size_t workspace_bytes_ = 0;
};

// Global-norm clip in place; returns the pre-clip norm (Clip.cpp semantics; synchronises).
float clip_gradient_norm(const std::vector<autograd::Variable>& parameters, float max_norm);

} // namespace veda::optim
