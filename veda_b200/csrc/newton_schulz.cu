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
// products read hi (bf16 outputs), or hi lo + lo hi + hi hi (fp32 outputs, errors of order 2^-20)
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
    CUtensorMap out;         // what the launch writes, in boxes of 32 x 32
    CUtensorMap out_t;       // S, P: the same for transposed tiles; kMuon: the bf16 weights
    int kind, tall, planes;
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
    int vec;                 // kOut, kMuon: the destination is stored by TMA
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
        int kbs, b, mb, nb;
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
        t.kbs = (k + pair::kBK - 1) / pair::kBK;
        t.a_mn = p.kind == kGram && p.tall;
        t.b_mn = p.kind == kGram ? p.tall != 0 : p.kind == kPoly ? false : p.tall == 0;
        t.idesc = pair::idesc(false, t.a_mn, t.b_mn);
        return true;
    }

    static __device__ __forceinline__ void operands(const Params& p, const Tile& t, int rank, int k, int za,
                                                    int zb, pair::Piece& a, pair::Piece& b)
    {
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

    // Epilogue staging. A warp takes 32 rows x 128 columns in four chunks of 32 columns through 8 KB
    // of shared memory: what a chunk needs of X or S (and the weights) is copied in asynchronously,
    // coalesced, before the tile's products are done; each lane then works on its row in place, and
    // the chunk leaves by TMA. Read directly by each lane from its own row, the same epilogues made
    // the products wait (a X + P X of 28 x 2048 x 1024: 195 us; the weights' update 1860 us).
    //   offset 0    hi tile (32 rows x 64 bytes, 64-byte swizzle); out: hi, bf16 result, bf16 weights
    //          2 K  lo tile; out: lo (for unsplit S and P: the transposed tile)
    //          4 K  fp32 weights (32 rows x 128 bytes, 128-byte swizzle); split S and P: transposed
    //               hi and lo; fp32 results take 0 .. 4 K
    // Where a chunk needs 4 KB, two sets alternate.
    static constexpr int kChunk = 32;
    static constexpr int kHalfTile = 32 * 64;
    static __device__ __forceinline__ int sets(const Params& p)
    {
        return p.kind == kMuon || (p.kind <= kPoly && p.planes > 1) ? 1 : 2;
    }
    static __device__ __forceinline__ uint32_t swz64(int r, int s)
    {
        return static_cast<uint32_t>(r * 64 + ((s ^ ((r >> 1) & 3)) << 4));
    }
    static __device__ __forceinline__ void copy16(void* dst, const void* src, bool in)
    {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(dst)), "l"(src),
                     "r"(in ? 16u : 0u)
                     : "memory");
    }
    // 32 rows x 32 16-bit columns of a plane; zeros past the last row and column
    static __device__ __forceinline__ void copy_plane(uint8_t* tile, const uint16_t* src, int64_t ld, int row, int col,
                                                      int nrows, int ncols, int lane)
    {
        const int seg = lane & 3, c = col + seg * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const int r = 8 * k + (lane >> 2);
            const bool in = row + r < nrows && c < ncols;
            copy16(tile + swz64(r, seg), in ? src + (row + r) * ld + c : src, in);
        }
    }

    // Starts the copies of chunk j into its set, one group per chunk (empty where nothing is read).
    static __device__ __forceinline__ void load_chunk(const Params& p, const Tile& t, int j, int trow, int tcol,
                                                      uint8_t* stage, int lane)
    {
        uint8_t* set = stage + (sets(p) == 2 ? (j & 1) * 2 * kHalfTile : 0);
        const int col = tcol + j * kChunk;
        if (p.kind == kPoly)
        {
            const uint16_t* src = p.s + p.plane_s * p.planes * t.b;
            copy_plane(set, src, p.lds, trow, col, p.m, p.m, lane);
            if (p.planes > 1) copy_plane(set + kHalfTile, src + p.plane_s, p.lds, trow, col, p.m, p.m, lane);
        }
        else if (p.kind != kGram)
        {
            const uint16_t* src = p.xh + p.plane_x * 2 * t.b;
            copy_plane(set, src, p.ldx, trow, col, p.rows, p.cols, lane);
            copy_plane(set + kHalfTile, src + p.plane_x, p.ldx, trow, col, p.rows, p.cols, lane);
            if (p.kind == kMuon && p.vec)
            {
                const float* w = p.master + p.stride_o * t.b;
                const int seg = lane & 7, c = col + seg * 4;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    const int r = 4 * k + (lane >> 3);
                    const bool in = trow + r < p.rows && c < p.cols;
                    copy16(set + 2 * kHalfTile + tc::sw128_offset(r, seg), in ? w + (trow + r) * p.ldo + c : w, in);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    static __device__ __forceinline__ void before(const Params& p, const Tile& t, State&, int row0, int col0,
                                                  pair::Staging& st, int lane)
    {
        // the last tile's copies have landed and its stores have read the staging
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (lane == 0)
        {
            tc::bulk_wait_group_read<0>();
        }
        __syncwarp();
        const int n = sets(p);
        for (int j = 0; j < n; ++j)
        {
            load_chunk(p, t, j, t.mb * pair::kTile + row0, t.nb * pair::kTile + col0, st.base, lane);
        }
    }

    // v += f x the lane's row of a staged 16-bit tile
    static __device__ __forceinline__ void add_tile(const uint8_t* tile, int lane, float f, float (&v)[kChunk])
    {
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const uint4 q = *reinterpret_cast<const uint4*>(tile + swz64(lane, k));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const float2 e = unpack_f16(w[i]);
                v[8 * k + 2 * i] = fmaf(f, e.x, v[8 * k + 2 * i]);
                v[8 * k + 2 * i + 1] = fmaf(f, e.y, v[8 * k + 2 * i + 1]);
            }
        }
    }
    static __device__ __forceinline__ void put_tile(uint8_t* tile, int lane, const uint32_t (&w)[16])
    {
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            *reinterpret_cast<uint4*>(tile + swz64(lane, k)) =
                make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        }
    }
    // the same transposed: tile row = column, tile column = lane, no swizzle (64 contiguous bytes a store)
    static __device__ __forceinline__ void put_transposed(uint8_t* tile, int lane, const uint32_t (&w)[16])
    {
        uint16_t* out = reinterpret_cast<uint16_t*>(tile) + lane;
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            out[(2 * i) * 32] = static_cast<uint16_t>(w[i] & 0xFFFFu);
            out[(2 * i + 1) * 32] = static_cast<uint16_t>(w[i] >> 16);
        }
    }

    template <int COLS>
    static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, State&, uint32_t taddr,
                                                    int row0, int col0, pair::Staging& st, int lane)
    {
        const int trow = t.mb * pair::kTile + row0, tcol = t.nb * pair::kTile + col0;
        const bool sym = p.kind <= kPoly;
        const int nrows = sym ? p.m : p.rows, ncols = sym ? p.m : p.cols;
        if (trow >= nrows || (p.kind == kMuon && skipped_step(p.flags, p.sumsq, p.grad_scale)))
        {
            return;
        }
        const int row = trow + lane;
        const int nsets = sets(p);
        const bool mirror = sym && t.mb != t.nb;
        // the tile's sums carry kUnit^2; what is stored carries kUnit
        const float f = (p.kind == kPoly ? p.cc : 1.0f) / kUnit;
        const float g = p.kind == kPoly ? p.cb : p.ca;
#pragma unroll 1
        for (int j = 0; j < COLS / kChunk; ++j)
        {
            const int col = tcol + j * kChunk;
            if (col >= ncols)
            {
                break;
            }
            uint8_t* set = st.base + (nsets == 2 ? (j & 1) * 2 * kHalfTile : 0);
            if (p.kind == kGram)
            {
                // nothing is copied in: the stores of the chunk that last used the set have read it
                if (lane == 0)
                {
                    nsets == 2 ? tc::bulk_wait_group_read<1>() : tc::bulk_wait_group_read<0>();
                }
            }
            else if (nsets == 2)
            {
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            }
            else
            {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncwarp();
            uint32_t r[kChunk];
            tc::tmem_ld32(taddr + static_cast<uint32_t>(j * kChunk), r);
            float v[kChunk];
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[i] = __uint_as_float(r[i]) * f;
            if (p.kind != kGram)
            {
                // lo first: the smaller addend
                if (!sym || p.planes > 1) add_tile(set + kHalfTile, lane, g, v);
                add_tile(set, lane, g, v);
            }
            if (p.kind == kOut || p.kind == kMuon)
            {
                finish(p, t, row, col, ncols - col, row < nrows, set, lane, v);
            }
            else
            {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    hi[i] = pack_f16(v[2 * i], v[2 * i + 1]);
                    const float2 h = unpack_f16(hi[i]);
                    lo[i] = pack_f16(v[2 * i] - h.x, v[2 * i + 1] - h.y);
                }
                const int planes = sym ? p.planes : 2, z = planes * t.b;
                put_tile(set, lane, hi);
                if (planes > 1) put_tile(set + kHalfTile, lane, lo);
                if (mirror)
                {
                    put_transposed(set + planes * kHalfTile, lane, hi);
                    if (planes > 1) put_transposed(set + 3 * kHalfTile, lane, lo);
                }
                tc::fence_proxy_async();
                __syncwarp();
                if (lane == 0)
                {
                    tc::tma_store_3d(&p.out, set, col, trow, z);
                    if (planes > 1) tc::tma_store_3d(&p.out, set + kHalfTile, col, trow, z + 1);
                    if (mirror)
                    {
                        tc::tma_store_3d(&p.out_t, set + planes * kHalfTile, trow, col, z);
                        if (planes > 1) tc::tma_store_3d(&p.out_t, set + 3 * kHalfTile, trow, col, z + 1);
                    }
                    tc::bulk_commit_group();
                }
            }
            if (p.kind != kGram)
            {
                if (j + nsets < COLS / kChunk)
                {
                    if (lane == 0)
                    {
                        tc::bulk_wait_group_read<0>();   // the set's stores have read it
                    }
                    __syncwarp();
                    load_chunk(p, t, j + nsets, trow, tcol, st.base, lane);
                }
                else
                {
                    asm volatile("cp.async.commit_group;" ::: "memory");   // keeps the group count
                }
            }
        }
    }

    // The last product's result: written out, or applied to the weights, through the staged tiles
    // where TMA can describe the destination (vec), else element by element.
    static __device__ __forceinline__ void finish(const Params& p, const Tile& t, int row, int col, int left, bool in,
                                                  uint8_t* set, int lane, float (&v)[kChunk])
    {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) v[i] *= 1.0f / kUnit;
        const int64_t at = p.stride_o * t.b + static_cast<int64_t>(row) * p.ldo + col;
        if (p.kind == kMuon)
        {
            uint8_t* tile = set + 2 * kHalfTile;
            if (p.vec)
            {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    float4* w4 = reinterpret_cast<float4*>(tile + tc::sw128_offset(lane, k));
                    float4 w = *w4;
                    v[4 * k] = update(p, w.x, v[4 * k]);
                    v[4 * k + 1] = update(p, w.y, v[4 * k + 1]);
                    v[4 * k + 2] = update(p, w.z, v[4 * k + 2]);
                    v[4 * k + 3] = update(p, w.w, v[4 * k + 3]);
                    *w4 = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                }
            }
            else if (in)
            {
#pragma unroll
                for (int i = 0; i < kChunk; ++i)
                {
                    if (i < left)
                    {
                        v[i] = update(p, p.master[at + i], v[i]);
                        p.master[at + i] = v[i];
                        if (p.lowp != nullptr) p.lowp[at + i] = __float2bfloat16_rn(v[i]);
                    }
                }
            }
        }
        else if (p.out_f32 && p.vec)
        {
            __syncwarp();   // every lane has read its row of the tiles that the result overwrites
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                *reinterpret_cast<float4*>(set + tc::sw128_offset(lane, k)) =
                    make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            }
        }
        if (!p.vec)
        {
            if (p.kind == kOut && in)
            {
#pragma unroll
                for (int i = 0; i < kChunk; ++i)
                {
                    if (i < left)
                    {
                        if (p.out_f32) static_cast<float*>(p.dst)[at + i] = v[i];
                        else static_cast<bf16*>(p.dst)[at + i] = __float2bfloat16_rn(v[i]);
                    }
                }
            }
            __syncwarp();   // the tiles may be loaded again
            return;
        }
        const bool half = p.kind == kMuon ? p.lowp != nullptr : !p.out_f32;
        if (half)
        {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            put_tile(set, lane, w);
        }
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0)
        {
            const int trow = row - lane;
            if (p.kind == kMuon) tc::tma_store_3d(&p.out, set + 2 * kHalfTile, col, trow, t.b);
            else tc::tma_store_3d(&p.out, set, col, trow, t.b);
            if (p.kind == kMuon && half) tc::tma_store_3d(&p.out_t, set, col, trow, t.b);
            tc::bulk_commit_group();
        }
    }

    static __device__ __forceinline__ float update(const Params& p, float w, float o)
    {
        w = __fsub_rn(w, __fmul_rn(p.decay, w));
        return __fsub_rn(w, __fmul_rn(p.step, o));
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
__device__ __forceinline__ float seen(float g, float scale, float clip)
{
    if (scale != 1.0f) g = __fmul_rn(g, scale);
    if (clip != 1.0f) g = __fmul_rn(g, clip);
    return g;
}

// N elements at p: one vector load when N > 1
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N])
{
    if constexpr (N == 1) v[0] = to_f32(*p);
    else if constexpr (sizeof(T) == 4)
    {
        const float4 q = *reinterpret_cast<const float4*>(p);
        v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
    }
    else
    {
        const uint2 q = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(q.x << 16), v[1] = __uint_as_float(q.x & 0xFFFF0000u);
        v[2] = __uint_as_float(q.y << 16), v[3] = __uint_as_float(q.y & 0xFFFF0000u);
    }
}

// A block takes every gridDim.x-th group of eight rows of matrix blockIdx.y, a warp a row, N elements
// a lane at a time (4 where rows and bases allow 16-byte accesses of fp32).
// Updates the momentum (Muon) and leaves the block's sum of squares of what is orthogonalised: G, the
// momentum m <- beta m + g, or g + beta m (Nesterov). Sums in double: fp32 squares overflow at 2^64.
template <typename T, int N>
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
    const T* g = static_cast<const T*>(s.g);
    double total = 0.0;
    for (int r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8)
    {
        const int64_t base = s.stride * blockIdx.y + r * s.ld;
#pragma unroll 4
        for (int c = (threadIdx.x & 31) * N; c < cols; c += 32 * N)
        {
            float u[N];
            load_n<T, N>(g + base + c, u);
            if (s.momentum != nullptr)
            {
                float m[N];
                load_n<float, N>(s.momentum + base + c, m);
#pragma unroll
                for (int k = 0; k < N; ++k)
                {
                    u[k] = seen(u[k], s.grad_scale, clip);
                    m[k] = fmaf(s.beta, m[k], u[k]);
                    u[k] = s.nesterov ? fmaf(s.beta, m[k], u[k]) : m[k];
                }
                if constexpr (N == 4) *reinterpret_cast<float4*>(s.momentum + base + c) = make_float4(m[0], m[1], m[2], m[3]);
                else s.momentum[base + c] = m[0];
            }
#pragma unroll
            for (int k = 0; k < N; ++k) total += static_cast<double>(u[k]) * u[k];
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

// X's two planes: 1024 u / (|u| + eps), the norm summed from the blocks' partials in a fixed order.
template <typename T, int N>
__global__ void __launch_bounds__(256)
init_kernel(Source s, int rows, int cols, const double* __restrict__ partials, float eps, uint16_t* __restrict__ x,
            int64_t ldx, int64_t plane)
{
    __shared__ double part[8];
    dep_wait();
    dep_release();
    if (skipped_step(s.flags, s.sumsq, s.grad_scale))
    {
        return;
    }
    // at most 256 blocks a matrix
    double total = threadIdx.x < gridDim.x ? partials[blockIdx.y * gridDim.x + threadIdx.x] : 0.0;
    total = warp_sum(total);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = total;
    __syncthreads();
    total = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
    const float scale = static_cast<float>(static_cast<double>(kUnit) / (sqrt(total) + static_cast<double>(eps)));
    const float clip = clip_scale(s.sumsq, s.max_norm, s.grad_scale);
    const T* g = static_cast<const T*>(s.g);
    for (int r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8)
    {
        const int64_t base = s.stride * blockIdx.y + r * s.ld;
        uint16_t* out = x + plane * 2 * blockIdx.y + r * ldx;
#pragma unroll 4
        for (int c = (threadIdx.x & 31) * N; c < cols; c += 32 * N)
        {
            float u[N];
            if (s.momentum == nullptr || s.nesterov)
            {
                load_n<T, N>(g + base + c, u);
            }
            if (s.momentum != nullptr)
            {
                float m[N];
                load_n<float, N>(s.momentum + base + c, m);
#pragma unroll
                for (int k = 0; k < N; ++k)
                {
                    u[k] = s.nesterov ? fmaf(s.beta, m[k], seen(u[k], s.grad_scale, clip)) : m[k];
                }
            }
            uint16_t hi[N], lo[N];
#pragma unroll
            for (int k = 0; k < N; ++k)
            {
                const float v = u[k] * scale;
                const __half h = __float2half_rn(v);
                hi[k] = __half_as_ushort(h);
                lo[k] = __half_as_ushort(__float2half_rn(v - __half2float(h)));
            }
            if constexpr (N == 4)
            {
                *reinterpret_cast<uint2*>(out + c) = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
                *reinterpret_cast<uint2*>(out + plane + c) = make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
            }
            else
            {
                out[c] = hi[0];
                out[plane + c] = lo[0];
            }
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
    // 8 rows a pass, at most 256 blocks a matrix; the same for every batch, so that a matrix's norm is
    l.blocks = static_cast<unsigned>(std::min<int64_t>((rows + 7) / 8, 256));
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
    const int clusters =
        split ? pair::clusters_available<Work, 8, true>() : pair::clusters_available<Work, 8, false>();
    if (clusters < 1)
    {
        return fail(VEDA_ERR_UNSUPPORTED, std::string(what) + ": no CTA pair fits on this device");
    }
    double* partials = reinterpret_cast<double*>(ws + l.partials);
    uint16_t* x[2] = {reinterpret_cast<uint16_t*>(ws + l.x[0]), reinterpret_cast<uint16_t*>(ws + l.x[1])};
    uint16_t* s = reinterpret_cast<uint16_t*>(ws + l.s);
    uint16_t* q = reinterpret_cast<uint16_t*>(ws + l.p);
    // tensor maps: X of either buffer (load, store), S and P (load, store, transposed store)
    CUtensorMap xl[2], xs[2], ml[2], ms[2], mt[2], dst{}, dst_low{};
    bool ok = true;
    for (int k = 0; k < 2; ++k)
    {
        ok = ok && pair::make_map3(&xl[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 64, 64) &&
             pair::make_map3(&xs[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 32, 32,
                             pair::Swizzle::k64);
        const uint16_t* m = k == 0 ? s : q;
        ok = ok && pair::make_map3(&ml[k], m, 2, false, l.m, l.m, l.planes * batch, l.lds, l.plane_s, 64, 64) &&
             pair::make_map3(&ms[k], m, 2, false, l.m, l.m, l.planes * batch, l.lds, l.plane_s, 32, 32,
                             pair::Swizzle::k64) &&
             pair::make_map3(&mt[k], m, 2, false, l.m, l.m, l.planes * batch, l.lds, l.plane_s, 32, 32,
                             pair::Swizzle::kNone);
    }
    if (!ok)
    {
        return fail(VEDA_ERR_CUDA, std::string(what) + ": tensor map creation failed");
    }
    // the destination by TMA where its base, pitch and stride are multiples of 16 bytes
    const auto fits = [&](const void* base, int es) {
        return aligned16(base) && p.ldo * es % 16 == 0 && (batch == 1 || p.stride_o * es % 16 == 0);
    };
    const int64_t stride = batch == 1 ? rows * p.ldo : p.stride_o;
    if (last == kMuon)
    {
        p.vec = fits(p.master, 4) && (p.lowp == nullptr || fits(p.lowp, 2)) &&
                pair::make_map3(&dst, p.master, 4, false, cols, rows, batch, p.ldo, stride, 32, 32) &&
                (p.lowp == nullptr || pair::make_map3(&dst_low, p.lowp, 2, true, cols, rows, batch, p.ldo, stride, 32,
                                                      32, pair::Swizzle::k64));
    }
    else
    {
        const int es = p.out_f32 ? 4 : 2;
        p.vec = fits(p.dst, es) && pair::make_map3(&dst, p.dst, es, !p.out_f32, cols, rows, batch, p.ldo, stride, 32, 32,
                                                   p.out_f32 ? pair::Swizzle::k128 : pair::Swizzle::k64);
    }
    const dim3 grid(l.blocks, static_cast<unsigned>(batch));
    // four elements at a time where every row of every matrix allows it
    const uintptr_t bases = reinterpret_cast<uintptr_t>(src.g) | reinterpret_cast<uintptr_t>(src.momentum);
    const bool four = (bases & (src.momentum != nullptr ? 15u : 4 * sizeof(T) - 1)) == 0 && cols % 4 == 0 &&
                      src.ld % 4 == 0 && (batch == 1 || src.stride % 4 == 0);
    int rc = launch(what, four ? norm_kernel<T, 4> : norm_kernel<T, 1>, grid, dim3(256), 0, stream, src,
                    static_cast<int>(rows), static_cast<int>(cols), partials);
    if (rc != VEDA_OK) return rc;
    rc = launch(what, four ? init_kernel<T, 4> : init_kernel<T, 1>, grid, dim3(256), 0, stream, src,
                static_cast<int>(rows), static_cast<int>(cols), static_cast<const double*>(partials), eps, x[0], l.ldx,
                l.plane_x);
    if (rc != VEDA_OK) return rc;
    p.tall = rows > cols;
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
            p.out = step == 0 ? ms[0] : step == 1 ? ms[1] : k < steps - 1 ? xs[(k + 1) & 1] : dst;
            p.out_t = step == 0 ? mt[0] : step == 1 ? mt[1] : dst_low;
            const int64_t units = static_cast<int64_t>(p.tiles) * batch;
            if (units >= (1ll << 30))
            {
                return fail(VEDA_ERR_INVALID_ARGUMENT, std::string(what) + ": too many tiles");
            }
            const int grid = static_cast<int>(std::min<int64_t>(units, clusters));
            rc = split ? pair::launch_pair<Work, 8, true>(what, p, grid, stream)
                       : pair::launch_pair<Work, 8, false>(what, p, grid, stream);
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
