// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step built on it.
//
// For each matrix of a batch, X = G / (|G|_F + eps), then `steps` times
//   S = X X^T (of the smaller side),  P = b S + c S^2,  X <- a X + P X,
// the odd quintic a s + b s^3 + c s^5 applied to every singular value. Three products an iteration
// on the CTA-pair tensor-core kernel (pair_mma.cuh), the whole batch in one launch each; a tall
// matrix is multiplied from the other side (S = X^T X, X <- a X + X P) by operand order alone, so
// nothing is transposed. S and P are symmetric: the tiles on and above the diagonal are computed,
// and each one above it is written a second time, transposed.
//
// Precision. X is held as two fp16 values, 1024 X = hi + lo (22 bits), because the quintic's slope
// of 3.4 at 0 amplifies what is rounded off X some 480 times over five steps: with X in 16 bits
// alone, rounding noise grows into spurious directions (bf16: 1 % of the result on random matrices,
// a third of it on low-rank ones; fp16 with the lo half in the a X term: 0.15 % and 0.03 %). The
// products read hi (bf16 outputs), or hi hi + hi lo + lo hi (fp32 outputs, errors of order 2^-20)
// with three times the k-blocks. fp16, not bf16: the values are bounded (singular values stay below
// 1.3, entries of P below 8), so its 11 bits cost nothing in range; 1024 keeps entries of order
// 1 / n and their lo halves away from fp16's smallest step.
#include "clip.cuh"
#include "pair_mma.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace veda::cuda
{
int* device_status_ptr();

namespace ns
{

constexpr float kUnit = 1024.0f;   // stored value = kUnit x value

enum Kind { kGram, kPoly, kApply, kOut, kMuon };

struct Params
{
    CUtensorMap x;           // [cols, rows, 2 batch]: planes hi, lo of each matrix (64 x 64 boxes)
    CUtensorMap a, b;        // [m, m, planes batch]: S and P
    CUtensorMap out;         // store boxes (64 x 32) of what the launch writes
    CUtensorMap out_t;       // transposed store boxes (32 x 64) of the same
    int kind, tall, segments, planes;
    int rows, cols, m;
    int batch, tm, tn, tiles;   // tiles of 256 per matrix: tm x tn, or tm (tm + 1) / 2 symmetric ones
    float ca, cb, cc;
    const uint16_t* xh;      // X as read by the epilogue: planes, pitch and plane stride
    const uint16_t* s;       // S as read by the epilogue
    int64_t ldx, plane_x, lds, plane_s;
    // kOut
    void* dst;
    int64_t ldo, stride_o;
    int out_f32;
    // kMuon
    float* master;
    bf16* lowp;
    float decay, step;       // lr weight_decay, lr scale
    const double* sumsq;
    float grad_scale;
    int flags;
    int* status;
};

__device__ __forceinline__ uint32_t pack_f16(float a, float b)
{
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t w)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

struct Work
{
    using Params = ns::Params;
    struct Tile
    {
        bool skip, a_mn, b_mn;
        int kbs, per, b, mb, nb;
        uint32_t idesc;
    };
    struct State
    {
    };

    static __device__ __forceinline__ bool tile(const Params& p, int cid, int clusters, int i, Tile& t)
    {
        const int u = cid + i * clusters;
        if (u >= p.tiles * p.batch)
        {
            return false;
        }
        t.skip = false;
        t.b = u / p.tiles;
        int r = u - t.b * p.tiles;
        if (p.kind <= kPoly)
        {
            // row mb of the upper triangle holds tm - mb tiles
            t.mb = 0;
            while (r >= p.tm - t.mb)
            {
                r -= p.tm - t.mb;
                ++t.mb;
            }
            t.nb = t.mb + r;
        }
        else
        {
            t.mb = r / p.tn;
            t.nb = r - t.mb * p.tn;
        }
        const int k = p.kind == kGram ? (p.tall ? p.rows : p.cols) : p.m;
        t.per = (k + pair::kBK - 1) / pair::kBK;
        t.kbs = t.per * p.segments;
        t.a_mn = p.kind == kGram && p.tall;
        t.b_mn = p.kind == kGram ? p.tall != 0 : p.kind == kPoly ? false : p.tall == 0;
        t.idesc = pair::idesc(false, t.a_mn, t.b_mn);
        return true;
    }

    static __device__ __forceinline__ void operands(const Params& p, const Tile& t, int rank, int kb,
                                                    pair::Piece& a, pair::Piece& b)
    {
        const int seg = p.segments > 1 ? kb / t.per : 0;
        const int k = (kb - seg * t.per) * pair::kBK;
        const int za = seg == 2 ? 1 : 0, zb = seg == 1 ? 1 : 0;
        const int m = t.mb * pair::kTile + rank * 128, n = t.nb * pair::kTile + rank * 128;
        const int x0 = 2 * t.b, s0 = p.planes * t.b;
        if (p.kind == kGram)
        {
            a = p.tall ? pair::Piece{&p.x, m, k, x0 + za} : pair::Piece{&p.x, k, m, x0 + za};
            b = p.tall ? pair::Piece{&p.x, n, k, x0 + zb} : pair::Piece{&p.x, k, n, x0 + zb};
        }
        else if (p.kind == kPoly)
        {
            a = {&p.a, k, m, s0 + za};
            b = {&p.a, k, n, s0 + zb};
        }
        else if (p.tall)
        {
            a = {&p.x, k, m, x0 + za};
            b = {&p.b, k, n, s0 + zb};
        }
        else
        {
            a = {&p.b, k, m, s0 + za};
            b = {&p.x, n, k, x0 + zb};
        }
    }

    static __device__ __forceinline__ void before(const Params&, const Tile&, State&, int, int, int) {}

    // 64 columns of one plane's row as fp32 pairs, added to v (columns at or past `cols` left alone).
    static __device__ __forceinline__ void add_row(const uint16_t* src, int left, float f, float (&v)[64])
    {
        if (left >= 64)
        {
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                const uint4 q = reinterpret_cast<const uint4*>(src)[k];
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const float2 e = unpack_f16(w[j]);
                    v[8 * k + 2 * j] = fmaf(f, e.x, v[8 * k + 2 * j]);
                    v[8 * k + 2 * j + 1] = fmaf(f, e.y, v[8 * k + 2 * j + 1]);
                }
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < 64; ++j)
        {
            if (j < left)
            {
                v[j] = fmaf(f, __half2float(__ushort_as_half(src[j])), v[j]);
            }
        }
    }

    template <int COLS>
    static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, State&, uint32_t taddr,
                                                    int row0, int col0, pair::Staging& st, int lane)
    {
        const int trow = t.mb * pair::kTile + row0;
        const bool sym = p.kind <= kPoly;
        const int nrows = sym ? p.m : p.rows, ncols = sym ? p.m : p.cols;
        if (trow >= nrows)
        {
            return;
        }
        const int row = trow + lane;
        const bool in = row < nrows;
        if (p.kind == kMuon && skipped_step(p.flags, p.sumsq, p.grad_scale))
        {
            return;
        }
#pragma unroll 1
        for (int c = 0; c < COLS; c += 64)
        {
            const int col = t.nb * pair::kTile + col0 + c;
            const int left = ncols - col;
            if (left <= 0)
            {
                break;
            }
            uint32_t r0[32], r1[32];
            tc::tmem_ld32_async(taddr + static_cast<uint32_t>(c), r0);
            tc::tmem_ld32_async(taddr + static_cast<uint32_t>(c + 32), r1);
            tc::tmem_wait_ld();
            tc::reg_fence(r0);
            tc::reg_fence(r1);
            // the tile's sums carry kUnit^2; what is stored carries kUnit
            const float f = (p.kind == kPoly ? p.cc : 1.0f) / kUnit;
            float v[64];
#pragma unroll
            for (int j = 0; j < 32; ++j)
            {
                v[j] = __uint_as_float(r0[j]) * f;
                v[32 + j] = __uint_as_float(r1[j]) * f;
            }
            if (p.kind != kGram && in)
            {
                // lo first: the smaller addend
                const uint16_t* src = p.kind == kPoly ? p.s + p.plane_s * p.planes * t.b + row * p.lds + col
                                                      : p.xh + p.plane_x * 2 * t.b + row * p.ldx + col;
                const int64_t plane = p.kind == kPoly ? p.plane_s : p.plane_x;
                const float g = p.kind == kPoly ? p.cb : p.ca;
                if (p.kind != kPoly || p.planes > 1)
                {
                    add_row(src + plane, left, g, v);
                }
                add_row(src, left, g, v);
            }
            if (p.kind == kOut || p.kind == kMuon)
            {
                if (in)
                {
                    finish(p, t, row, col, left, v);
                }
                continue;
            }
            uint32_t hi[32], lo[32];
#pragma unroll
            for (int j = 0; j < 32; ++j)
            {
                hi[j] = pack_f16(v[2 * j], v[2 * j + 1]);
                const float2 h = unpack_f16(hi[j]);
                lo[j] = pack_f16(v[2 * j] - h.x, v[2 * j + 1] - h.y);
            }
            const int planes = p.kind == kApply ? 2 : p.planes;
            const int z = planes * t.b;
            send(p, hi, col, trow, z, st, lane);
            if (planes > 1)
            {
                send(p, lo, col, trow, z + 1, st, lane);
            }
            if (sym && t.mb != t.nb)
            {
                send_t(p, hi, col, trow, z, st, lane);
                if (planes > 1)
                {
                    send_t(p, lo, col, trow, z + 1, st, lane);
                }
            }
        }
    }

    static __device__ __forceinline__ void send(const Params& p, const uint32_t (&w)[32], int col, int row,
                                                int plane, pair::Staging& st, int lane)
    {
        uint8_t* buf = st.buffer(lane);
#pragma unroll
        for (int k = 0; k < 8; ++k)
        {
            *reinterpret_cast<uint4*>(buf + tc::sw128_offset(lane, k)) =
                make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        }
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0)
        {
            tc::tma_store_3d(&p.out, buf, col, row, plane);
            tc::bulk_commit_group();
        }
        st.sent();
    }

    // The same 32 rows x 64 columns at (col, row) transposed: a lane is a column of the 64 x 32 box.
    static __device__ __forceinline__ void send_t(const Params& p, const uint32_t (&w)[32], int col, int row,
                                                  int plane, pair::Staging& st, int lane)
    {
        uint16_t* buf = reinterpret_cast<uint16_t*>(st.buffer(lane));
#pragma unroll
        for (int j = 0; j < 32; ++j)
        {
            buf[(2 * j) * 32 + lane] = static_cast<uint16_t>(w[j] & 0xFFFFu);
            buf[(2 * j + 1) * 32 + lane] = static_cast<uint16_t>(w[j] >> 16);
        }
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0)
        {
            tc::tma_store_3d(&p.out_t, buf, row, col, plane);
            tc::bulk_commit_group();
        }
        st.sent();
    }

    // The last product's result: written out, or applied to the weights.
    static __device__ __forceinline__ void finish(const Params& p, const Tile& t, int row, int col, int left,
                                                  const float (&v)[64])
    {
        const int64_t at = p.stride_o * t.b + static_cast<int64_t>(row) * p.ldo + col;
#pragma unroll
        for (int j = 0; j < 64; ++j)
        {
            if (j < left)
            {
                const float o = v[j] / kUnit;
                if (p.kind == kMuon)
                {
                    float w = p.master[at + j];
                    w = __fsub_rn(w, __fmul_rn(p.decay, w));
                    w = __fsub_rn(w, __fmul_rn(p.step, o));
                    p.master[at + j] = w;
                    if (p.lowp != nullptr)
                    {
                        p.lowp[at + j] = __float2bfloat16_rn(w);
                    }
                }
                else if (p.out_f32)
                {
                    static_cast<float*>(p.dst)[at + j] = o;
                }
                else
                {
                    static_cast<bf16*>(p.dst)[at + j] = __float2bfloat16_rn(o);
                }
            }
        }
    }
};

// ---- what is orthogonalised, its norm, and X ----------------------------------------------------
struct Source
{
    const void* g;           // a matrix per stride elements, rows of pitch ld
    int64_t ld, stride;
    float* momentum;         // Muon: updated in place (pitch and stride as g's), else null
    float beta;
    int nesterov;
    const double* sumsq;
    float max_norm, grad_scale;
    int flags;
};

// The gradient as the step sees it: scaled and clipped.
template <typename T>
__device__ __forceinline__ float gradient(const Source& s, int64_t at, float scale, float clip)
{
    float g = to_f32(static_cast<const T*>(s.g)[at]);
    if (scale != 1.0f) g = __fmul_rn(g, scale);
    if (clip != 1.0f) g = __fmul_rn(g, clip);
    return g;
}

// One block of a matrix's rows: updates the momentum (Muon) and leaves the block's sum of squares of
// what is orthogonalised: G, the momentum m <- beta m + g, or g + beta m (Nesterov).
template <typename T>
__global__ void __launch_bounds__(256)
norm_kernel(Source s, int rows, int cols, double* __restrict__ partials)
{
    __shared__ double part[8];
    dep_wait();
    dep_release();
    if (skipped_step(s.flags, s.sumsq, s.grad_scale))
    {
        return;
    }
    const float clip = clip_scale(s.sumsq, s.max_norm, s.grad_scale);
    double total = 0.0;
    for (int r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8)
    {
        const int64_t base = s.stride * blockIdx.y + r * s.ld;
        for (int c = threadIdx.x & 31; c < cols; c += 32)
        {
            float u = gradient<T>(s, base + c, s.grad_scale, clip);
            if (s.momentum != nullptr)
            {
                const float m = fmaf(s.beta, s.momentum[base + c], u);
                s.momentum[base + c] = m;
                u = s.nesterov ? fmaf(s.beta, m, u) : m;
            }
            total += static_cast<double>(u) * u;
        }
    }
    total = warp_sum(total);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = total;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        for (int k = 1; k < 8; ++k) total += part[k];
        partials[blockIdx.y * gridDim.x + blockIdx.x] = total;
    }
}

// X's two planes: 1024 u / (|u| + eps), the norm summed from the blocks' partials in order.
template <typename T>
__global__ void __launch_bounds__(256)
init_kernel(Source s, int rows, int cols, const double* __restrict__ partials, float eps, uint16_t* __restrict__ x,
            int64_t ldx, int64_t plane)
{
    __shared__ float scale_shared;
    dep_wait();
    dep_release();
    if (skipped_step(s.flags, s.sumsq, s.grad_scale))
    {
        return;
    }
    if (threadIdx.x == 0)
    {
        double total = 0.0;
        for (int k = 0; k < static_cast<int>(gridDim.x); ++k) total += partials[blockIdx.y * gridDim.x + k];
        scale_shared = static_cast<float>(static_cast<double>(kUnit) / (sqrt(total) + static_cast<double>(eps)));
    }
    __syncthreads();
    const float scale = scale_shared;
    const float clip = clip_scale(s.sumsq, s.max_norm, s.grad_scale);
    for (int r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8)
    {
        const int64_t base = s.stride * blockIdx.y + r * s.ld;
        uint16_t* out = x + plane * 2 * blockIdx.y + r * ldx;
        for (int c = threadIdx.x & 31; c < cols; c += 32)
        {
            float u;
            if (s.momentum != nullptr)
            {
                const float m = s.momentum[base + c];
                u = s.nesterov ? fmaf(s.beta, m, gradient<T>(s, base + c, s.grad_scale, clip)) : m;
            }
            else
            {
                u = gradient<T>(s, base + c, 1.0f, 1.0f);
            }
            const float v = u * scale;
            const __half h = __float2half_rn(v);
            out[c] = __half_as_ushort(h);
            out[plane + c] = __half_as_ushort(__float2half_rn(v - __half2float(h)));
        }
    }
}

// ---- host ------------------------------------------------------------------------------------
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

constexpr int64_t kMaxExtent = 1 << 20;
constexpr int64_t kMaxBatch = 1 << 15;

struct Layout
{
    int planes;              // of S and P: 1, or 2 for split products
    int64_t m, ldx, plane_x, lds, plane_s;
    unsigned blocks;         // per matrix, of the elementwise launches
    size_t partials, x[2], s, p, total;
};

Layout layout(int64_t batch, int64_t rows, int64_t cols, bool split)
{
    Layout l{};
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += static_cast<size_t>(round_up(bytes, 256));
        return here;
    };
    l.planes = split ? 2 : 1;
    l.m = std::min(rows, cols);
    l.ldx = round_up(cols, 8);
    l.plane_x = rows * l.ldx;
    l.lds = round_up(l.m, 8);
    l.plane_s = l.m * l.lds;
    // 8 rows a pass; enough blocks to fill the GPU four times over the batch, at most 64 a matrix
    const int64_t want = std::max<int64_t>(1, 4 * 148 / batch);
    l.blocks = static_cast<unsigned>(std::min<int64_t>({(rows + 7) / 8, want, 64}));
    l.partials = take(batch * l.blocks * 8);
    l.x[0] = take(batch * 2 * l.plane_x * 2);
    l.x[1] = take(batch * 2 * l.plane_x * 2);
    l.s = take(batch * l.planes * l.plane_s * 2);
    l.p = take(batch * l.planes * l.plane_s * 2);
    l.total = at;
    return l;
}

// norm, X, then the products of every step; p's output fields say what the last one writes.
template <typename T>
int iterate(const char* what, const Source& src, int64_t batch, int64_t rows, int64_t cols, int steps, float a,
            float b, float c, float eps, bool split, int last, char* ws, Params p, cudaStream_t stream)
{
    const Layout l = layout(batch, rows, cols, split);
    const int clusters = pair::clusters_available<Work, 4>();
    if (clusters < 1)
    {
        return fail(VEDA_ERR_UNSUPPORTED, std::string(what) + ": no CTA pair fits on this device");
    }
    double* partials = reinterpret_cast<double*>(ws + l.partials);
    uint16_t* x[2] = {reinterpret_cast<uint16_t*>(ws + l.x[0]), reinterpret_cast<uint16_t*>(ws + l.x[1])};
    uint16_t* s = reinterpret_cast<uint16_t*>(ws + l.s);
    uint16_t* q = reinterpret_cast<uint16_t*>(ws + l.p);
    // tensor maps: X of either buffer (load, store), S and P (load, store, transposed store)
    CUtensorMap xl[2], xs[2], ml[2], ms[2], mt[2];
    bool ok = true;
    for (int k = 0; k < 2; ++k)
    {
        ok = ok && pair::make_map3(&xl[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 64, 64) &&
             pair::make_map3(&xs[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 64, 32);
        const uint16_t* m = k == 0 ? s : q;
        ok = ok && pair::make_map3(&ml[k], m, 2, false, l.m, l.m, l.planes * batch, l.lds, l.plane_s, 64, 64) &&
             pair::make_map3(&ms[k], m, 2, false, l.m, l.m, l.planes * batch, l.lds, l.plane_s, 64, 32) &&
             pair::make_map3(&mt[k], m, 2, false, l.m, l.m, l.planes * batch, l.lds, l.plane_s, 32, 64, false);
    }
    if (!ok)
    {
        return fail(VEDA_ERR_CUDA, std::string(what) + ": tensor map creation failed");
    }
    const dim3 grid(l.blocks, static_cast<unsigned>(batch));
    int rc = launch(what, norm_kernel<T>, grid, dim3(256), 0, stream, src, static_cast<int>(rows),
                    static_cast<int>(cols), partials);
    if (rc != VEDA_OK) return rc;
    rc = launch(what, init_kernel<T>, grid, dim3(256), 0, stream, src, static_cast<int>(rows),
                static_cast<int>(cols), static_cast<const double*>(partials), eps, x[0], l.ldx, l.plane_x);
    if (rc != VEDA_OK) return rc;
    p.tall = rows > cols;
    p.segments = split ? 3 : 1;
    p.planes = l.planes;
    p.rows = static_cast<int>(rows);
    p.cols = static_cast<int>(cols);
    p.m = static_cast<int>(l.m);
    p.batch = static_cast<int>(batch);
    p.ca = a;
    p.cb = b;
    p.cc = c;
    p.s = s;
    p.ldx = l.ldx;
    p.plane_x = l.plane_x;
    p.lds = l.lds;
    p.plane_s = l.plane_s;
    p.a = ml[0];
    p.b = ml[1];
    p.status = device_status_ptr();
    const int tm = static_cast<int>((l.m + 255) / 256);
    for (int k = 0; k < steps; ++k)
    {
        p.x = xl[k & 1];
        p.xh = x[k & 1];
        for (int step = 0; step < 3; ++step)
        {
            p.kind = step < 2 ? step : k == steps - 1 ? last : kApply;
            p.tm = step < 2 ? tm : static_cast<int>((rows + 255) / 256);
            p.tn = step < 2 ? tm : static_cast<int>((cols + 255) / 256);
            p.tiles = step < 2 ? tm * (tm + 1) / 2 : p.tm * p.tn;
            p.out = step == 0 ? ms[0] : step == 1 ? ms[1] : xs[(k + 1) & 1];
            p.out_t = step == 0 ? mt[0] : mt[1];
            const int64_t units = static_cast<int64_t>(p.tiles) * batch;
            if (units >= (1ll << 30))
            {
                return fail(VEDA_ERR_INVALID_ARGUMENT, std::string(what) + ": too many tiles");
            }
            rc = pair::launch_pair<Work, 4>(what, p, static_cast<int>(std::min<int64_t>(units, clusters)), stream);
            if (rc != VEDA_OK) return rc;
        }
    }
    return VEDA_OK;
}

bool bad_extent(int64_t batch, int64_t rows, int64_t cols)
{
    return batch < 0 || rows < 0 || cols < 0 || batch > kMaxBatch || rows > kMaxExtent || cols > kMaxExtent;
}

int check_workspace(const char* what, void* ws, size_t bytes, size_t want)
{
    if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255u) != 0 || bytes < want)
    {
        return fail(VEDA_ERR_INVALID_ARGUMENT,
                    std::string(what) + ": workspace too small or not 256-byte aligned (see " + what + "_workspace)");
    }
    return VEDA_OK;
}

} // namespace ns
} // namespace veda::cuda

using namespace veda::cuda;

extern "C" size_t veda_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols, int dtype)
{
    if (ns::bad_extent(batch, rows, cols) || batch == 0 || rows == 0 || cols == 0 || !valid_dtype(dtype))
    {
        return 0;
    }
    return ns::layout(batch, rows, cols, dtype == VEDA_F32).total;
}

extern "C" size_t veda_muon_step_workspace(int64_t batch, int64_t rows, int64_t cols, int dtype)
{
    return veda_orthogonalize_workspace(batch, rows, cols, dtype);
}

extern "C" int veda_orthogonalize(const void* g, int64_t ldg, int64_t stride_g, void* out, int64_t ldo,
                                  int64_t stride_o, int64_t batch, int64_t rows, int64_t cols, int steps, float a,
                                  float b, float c, float eps, void* workspace, size_t workspace_bytes, int dtype,
                                  veda_stream_t stream)
{
    VEDA_REQUIRE(valid_dtype(dtype), "unknown dtype");
    VEDA_REQUIRE(!ns::bad_extent(batch, rows, cols), "bad shape");
    VEDA_REQUIRE(ldg >= cols && ldo >= cols, "leading dimension smaller than cols");
    VEDA_REQUIRE(batch <= 1 || (stride_g >= 0 && stride_o >= (rows - 1) * ldo + cols),
                 "the matrices of the output overlap");
    VEDA_REQUIRE(steps >= 1, "at least one step");
    VEDA_REQUIRE(eps >= 0.0f, "eps must not be negative");
    if (batch == 0 || rows == 0 || cols == 0)
    {
        return VEDA_OK;
    }
    VEDA_REQUIRE(g != nullptr && out != nullptr, "null pointer");
    const bool split = dtype == VEDA_F32;
    int rc = ns::check_workspace("veda_orthogonalize", workspace, workspace_bytes,
                                 ns::layout(batch, rows, cols, split).total);
    if (rc != VEDA_OK) return rc;
    ns::Params p{};
    p.dst = out;
    p.ldo = ldo;
    p.stride_o = stride_o;
    p.out_f32 = split;
    const ns::Source src{g, ldg, stride_g, nullptr, 0.0f, 0, nullptr, 1.0f, 1.0f, 0};
    char* ws = static_cast<char*>(workspace);
    return split ? ns::iterate<float>("veda_orthogonalize", src, batch, rows, cols, steps, a, b, c, eps, true, ns::kOut,
                                      ws, p, stream)
                 : ns::iterate<bf16>("veda_orthogonalize", src, batch, rows, cols, steps, a, b, c, eps, false, ns::kOut,
                                     ws, p, stream);
}

extern "C" int veda_muon_step(float* master, float* momentum, const float* grad, void* lowp, int64_t batch,
                              int64_t rows, int64_t cols, int64_t stride, float lr, float beta, int nesterov,
                              float weight_decay, float update_scale, int steps, float a, float b, float c, float eps,
                              const double* sumsq, float max_norm, float grad_scale, int flags, void* workspace,
                              size_t workspace_bytes, veda_stream_t stream)
{
    VEDA_REQUIRE(!ns::bad_extent(batch, rows, cols), "bad shape");
    VEDA_REQUIRE(batch <= 1 || stride >= rows * cols, "the matrices overlap");
    VEDA_REQUIRE(lr >= 0.0f && eps >= 0.0f && weight_decay >= 0.0f,
                 "learning rate, eps and weight decay must not be negative");
    VEDA_REQUIRE(beta >= 0.0f && beta < 1.0f, "beta must lie in [0, 1)");
    VEDA_REQUIRE(sumsq == nullptr || max_norm > 0.0f, "max_norm must be positive");
    VEDA_REQUIRE(steps >= 1, "at least one step");
    if (batch == 0 || rows == 0 || cols == 0)
    {
        return VEDA_OK;
    }
    VEDA_REQUIRE(master != nullptr && momentum != nullptr && grad != nullptr, "null pointer");
    const bool split = lowp == nullptr;
    int rc = ns::check_workspace("veda_muon_step", workspace, workspace_bytes,
                                 ns::layout(batch, rows, cols, split).total);
    if (rc != VEDA_OK) return rc;
    ns::Params p{};
    p.master = master;
    p.lowp = static_cast<bf16*>(lowp);
    p.ldo = cols;
    p.stride_o = stride;
    p.decay = lr * weight_decay;
    p.step = lr * update_scale;
    p.sumsq = sumsq;
    p.grad_scale = grad_scale;
    p.flags = flags;
    const ns::Source src{grad, cols, stride, momentum, beta, nesterov, sumsq, max_norm, grad_scale, flags};
    return ns::iterate<float>("veda_muon_step", src, batch, rows, cols, steps, a, b, c, eps, split, ns::kMuon,
                              static_cast<char*>(workspace), p, stream);
}
