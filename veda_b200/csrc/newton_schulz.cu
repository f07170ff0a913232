// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step built on it.
//
// For each matrix of a batch, X = G / (|G|_F + eps), then `steps` times
//   S = X X^T (of the smaller side),  M = a I + b S + c S^2,  X <- M X,
// the odd quintic a s + b s^3 + c s^5 applied to every singular value. Three products an iteration
// on the CTA-pair tensor-core kernel (pair_mma.cuh), the whole batch in one launch each; a tall
// matrix is multiplied from the other side (S = X^T X, X <- X M) by operand order alone, so nothing
// is transposed. S and M are symmetric: the tiles on and above the diagonal are computed, and each
// one above it is written a second time, transposed.
//
// Precision. X is held as two fp16 values, 1024 X = hi + lo (22 bits), because the quintic's slope
// of 3.4 at 0 amplifies what is rounded off X some 480 times over five steps: with X in 16 bits
// alone, rounding noise grows into spurious directions (errors, relative to the result, on random /
// rank-8 matrices of 512 x 1024: bf16 1.0 % / 32 %; fp16 0.14 % / 4 %). For bf16 results the products
// read hi, and a lo, exact to first order where the slope matters, is added to them: 0.15 % / 0.13 %,
// less than the result's own rounding. Because M multiplies X as a whole, rounding M leaves the rank
// of X as it is. For fp32 results S, M and X enter as hi lo + lo hi + hi hi (errors of order 2^-20).
// fp16, not bf16: the values are bounded (singular values stay below 1.3, entries of M below 8), so
// its 11 bits cost nothing in range; 1024 keeps entries of order 1 / n and their lo halves away from
// fp16's smallest step.
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

// What a launch computes: S, M, the next X, or the last X as a result or as the weights' update.
enum Kind { kGram, kPoly, kApply, kOut, kMuon };

struct Params
{
    CUtensorMap a, b;        // operands: planes hi, lo of each matrix (X; S and M when split)
    CUtensorMap out;         // what the launch writes, in boxes of 32 x 32
    CUtensorMap out_t;       // S, M: the same for transposed tiles; kMuon: the bf16 weights
    int tall;
    int rows, cols;          // of X
    int nrows, ncols;        // of what is written
    int k;                   // terms of a sum
    int planes_a, planes_b;  // planes of a matrix in a and b
    int total, tm;           // tiles in all; kGram, kPoly: tiles of a side
    pair::Divisor per_matrix, by_n;
    float ca, cb, cc;
    const uint16_t* src;     // kPoly: S; later kinds: X (read by the epilogue)
    int64_t ld, plane;       // its pitch and plane stride
    // kOut, kMuon: the destination, stored by TMA if vec
    void* dst;               // kMuon: the fp32 weights
    int64_t ldo, stride_o;
    int out_f32, vec;
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

template <int KIND, bool SPLIT>
struct Work
{
    using Params = ns::Params;
    static constexpr bool SYM = KIND <= kPoly;
    struct Tile
    {
        bool skip, a_mn, b_mn;
        int kbs, b, mb, nb;
        uint32_t idesc;
    };
    struct State
    {
        int sent = 0;   // chunks written out so far: the output sets take turns by it across tiles
    };

    static __device__ __forceinline__ bool tile(const Params& p, int cid, int clusters, int i, Tile& t)
    {
        const int u = cid + i * clusters;
        if (u >= p.total)
        {
            return false;
        }
        int r;
        t.b = p.per_matrix.div(u, r);
        if constexpr (SYM)
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
            t.mb = p.by_n.div(r, t.nb);
        }
        t.skip = false;
        t.kbs = (p.k + pair::kBK - 1) / pair::kBK;
        // tall: S = X^T X, X M; else S = X X^T, M X; S and M read as they are, being symmetric
        t.a_mn = KIND == kGram && p.tall;
        t.b_mn = KIND == kGram ? p.tall != 0 : KIND != kPoly && p.tall == 0;
        t.idesc = pair::idesc(false, t.a_mn, t.b_mn);
        return true;
    }

    static __device__ __forceinline__ void operands(const Params& p, const Tile& t, int rank, pair::Piece& a,
                                                    pair::Piece& b)
    {
        const int m = t.mb * pair::kTile + rank * 128, n = t.nb * pair::kTile + rank * 128;
        a = {&p.a, t.a_mn ? m : 0, t.a_mn ? 0 : m, p.planes_a * t.b};
        b = {&p.b, t.b_mn ? n : 0, t.b_mn ? 0 : n, p.planes_b * t.b};
    }
    static __device__ __forceinline__ void prefetch(const Params& p)
    {
        tc::tma_prefetch(&p.a);
        tc::tma_prefetch(&p.b);
    }

    // Epilogue staging. A warp takes 32 rows x 128 columns in four chunks of 32 columns through 8 KB
    // of shared memory, four units of 2 KB (32 rows x 64 bytes, 64-byte swizzle) or two of 4 KB (32
    // rows x 128 bytes, 128-byte swizzle): what a chunk needs is copied in asynchronously, coalesced,
    // before the tile's products are done, each lane works on its row, and the chunk leaves by TMA.
    // Read and written by each lane in its own row of global memory instead, the epilogue held the
    // products up (M X of 28 x 2048 x 1024 195 us, the weights' update 1860 us).
    //                 copied in                     written out
    //   kGram         -                             hi, transposed hi, two sets
    //         split   -                             hi, lo, transposed hi, lo
    //   kPoly         S hi at 0 and 1 in turn       hi at 2, transposed at 3
    //         split   S hi at 0, lo at 1            hi, lo in place, transposed at 2 and 3
    //   kApply, kOut  X lo at 0 and 1 in turn       hi at 2, lo at 3; result at 2 and 3 in turn
    //         split   -                             hi, lo in two sets; fp32 result in two sets
    //   kMuon         X lo at 0, weights at 2 - 3   weights in place, bf16 weights at 1
    //         split   weights at 0 - 1, 2 - 3       in place
    static constexpr int kChunk = 32;
    static constexpr int kUnitBytes = 32 * 64;
    static constexpr bool READS_X = !SPLIT && !SYM;        // the a lo term
    static constexpr bool IN_PLACE = KIND == kMuon || (KIND == kPoly && SPLIT);
    // chunks copied in ahead, and sets that a chunk's output takes turns in
    static constexpr int AHEAD = KIND == kGram              ? 0
                                 : KIND == kPoly            ? (SPLIT ? 1 : 2)
                                 : KIND == kMuon            ? (SPLIT ? 2 : 1)
                                 : READS_X                  ? 2
                                                            : 0;
    static constexpr int OUTS = KIND == kGram    ? (SPLIT ? 1 : 2)
                                : KIND == kPoly  ? 1
                                : KIND == kApply ? (SPLIT ? 2 : 1)
                                                 : 2;
    static __device__ __forceinline__ int in_unit(int j)
    {
        return AHEAD == 2 ? (j & 1) * (KIND == kMuon ? 2 : 1) : 0;
    }
    static __device__ __forceinline__ int out_unit(int j)
    {
        if constexpr (KIND == kMuon) return 1;             // of the bf16 weights
        else if constexpr (KIND == kPoly) return SPLIT ? 0 : 2;
        else if constexpr (KIND == kGram) return SPLIT ? 0 : 2 * (j & 1);
        else if constexpr (SPLIT) return 2 * (j & 1);
        else return KIND == kOut ? 2 + (j & 1) : 2;
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
    static __device__ __forceinline__ void copy_plane(uint8_t* tile, const uint16_t* src, const Params& p, int row,
                                                      int col, int lane)
    {
        const int seg = lane & 3, c = col + seg * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const int r = 8 * k + (lane >> 2);
            const bool in = row + r < p.nrows && c < p.ncols;
            copy16(tile + swz64(r, seg), in ? src + (row + r) * p.ld + c : src, in);
        }
    }

    // Starts the copies of chunk j, one group (empty where nothing is read).
    static __device__ __forceinline__ void load_chunk(const Params& p, const Tile& t, int j, int trow, int tcol,
                                                      uint8_t* stage, int lane)
    {
        uint8_t* in = stage + in_unit(j) * kUnitBytes;
        const int col = tcol + j * kChunk;
        if constexpr (KIND == kPoly)
        {
            const uint16_t* src = p.src + p.plane * p.planes_a * t.b;
            copy_plane(in, src, p, trow, col, lane);
            if constexpr (SPLIT) copy_plane(in + kUnitBytes, src + p.plane, p, trow, col, lane);
        }
        if constexpr (READS_X)
        {
            copy_plane(in, p.src + p.plane * (2 * t.b + 1), p, trow, col, lane);
        }
        if constexpr (KIND == kMuon)
        {
            if (p.vec)
            {
                uint8_t* tile = SPLIT ? in : stage + 2 * kUnitBytes;
                const float* w = static_cast<const float*>(p.dst) + p.stride_o * t.b;
                const int seg = lane & 7, c = col + seg * 4;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    const int r = 4 * k + (lane >> 3);
                    const bool inside = trow + r < p.nrows && c < p.ncols;
                    copy16(tile + tc::sw128_offset(r, seg), inside ? w + (trow + r) * p.ldo + c : w, inside);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    static __device__ __forceinline__ void before(const Params& p, const Tile& t, State&, int row0, int col0,
                                                  pair::Staging& st, int lane)
    {
        if constexpr (AHEAD > 0)
        {
            // the last tile's copies have landed, and in place, its stores have read the staging
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (IN_PLACE && lane == 0)
            {
                tc::bulk_wait_group_read<0>();
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
            {
                load_chunk(p, t, j, t.mb * pair::kTile + row0, t.nb * pair::kTile + col0, st.base, lane);
            }
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
    static __device__ __forceinline__ void put_f32(uint8_t* tile, int lane, const float (&v)[kChunk])
    {
#pragma unroll
        for (int k = 0; k < 8; ++k)
        {
            *reinterpret_cast<float4*>(tile + tc::sw128_offset(lane, k)) =
                make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
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
    static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, State& s, uint32_t taddr,
                                                    int row0, int col0, pair::Staging& st, int lane)
    {
        const int trow = t.mb * pair::kTile + row0, tcol = t.nb * pair::kTile + col0;
        if (trow >= p.nrows || (KIND == kMuon && skipped_step(p.flags, p.sumsq, p.grad_scale)))
        {
            return;
        }
        const bool mirror = SYM && t.mb != t.nb;
        // the tile's sums carry kUnit^2; what is stored carries kUnit
        const float f = (KIND == kPoly ? p.cc : 1.0f) / kUnit;
#pragma unroll 1
        for (int j = 0; j < COLS / kChunk; ++j)
        {
            const int col = tcol + j * kChunk;
            if (col >= p.ncols)
            {
                break;
            }
            uint8_t* in = st.base + in_unit(j) * kUnitBytes;
            uint8_t* out = st.base + out_unit(s.sent++) * kUnitBytes;
            uint32_t r[kChunk];
            tc::tmem_ld32(taddr + static_cast<uint32_t>(j * kChunk), r);
            float v[kChunk];
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[i] = __uint_as_float(r[i]) * f;
            if constexpr (AHEAD > 0)
            {
                asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD > 0 ? AHEAD - 1 : 0) : "memory");
                __syncwarp();   // every lane's copies are visible to the warp
                if constexpr (KIND == kPoly)
                {
                    // lo first: the smaller addend
                    if constexpr (SPLIT) add_tile(in + kUnitBytes, lane, p.cb, v);
                    add_tile(in, lane, p.cb, v);
                }
                if constexpr (READS_X) add_tile(in, lane, p.ca, v);
            }
            if constexpr (KIND == kPoly)
            {
                const int d = trow + lane - col;   // the lane's diagonal element
#pragma unroll
                for (int i = 0; i < kChunk; ++i) v[i] = i == d ? v[i] + p.ca * kUnit : v[i];
            }
            if constexpr (!IN_PLACE)
            {
                if constexpr (AHEAD > 0)
                {
                    __syncwarp();   // the chunk is read: its unit is free
                    next_chunk<COLS>(p, t, j, trow, tcol, st.base, lane);
                }
                if (lane == 0)
                {
                    tc::bulk_wait_group_read<OUTS - 1>();   // the stores that last used `out` have read it
                }
                __syncwarp();
            }
            if constexpr (KIND == kOut || KIND == kMuon)
            {
                finish(p, t, trow, col, in, out, st.base, lane, v);
            }
            else
            {
                constexpr int PLANES = KIND == kApply || SPLIT ? 2 : 1;
                const int z = PLANES * t.b;
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    hi[i] = pack_f16(v[2 * i], v[2 * i + 1]);
                    if constexpr (PLANES == 2)
                    {
                        const float2 h = unpack_f16(hi[i]);
                        lo[i] = pack_f16(v[2 * i] - h.x, v[2 * i + 1] - h.y);
                    }
                }
                put_tile(out, lane, hi);
                if constexpr (PLANES == 2) put_tile(out + kUnitBytes, lane, lo);
                if (mirror)
                {
                    put_transposed(out + PLANES * kUnitBytes, lane, hi);
                    if constexpr (PLANES == 2) put_transposed(out + 3 * kUnitBytes, lane, lo);
                }
                tc::fence_proxy_async();
                __syncwarp();
                if (lane == 0)
                {
                    tc::tma_store_3d(&p.out, out, col, trow, z);
                    if constexpr (PLANES == 2) tc::tma_store_3d(&p.out, out + kUnitBytes, col, trow, z + 1);
                    if (mirror)
                    {
                        tc::tma_store_3d(&p.out_t, out + PLANES * kUnitBytes, trow, col, z);
                        if constexpr (PLANES == 2) tc::tma_store_3d(&p.out_t, out + 3 * kUnitBytes, trow, col, z + 1);
                    }
                    tc::bulk_commit_group();
                }
            }
            if constexpr (IN_PLACE)
            {
                if (lane == 0)
                {
                    tc::bulk_wait_group_read<0>();   // the stores have read the units
                }
                __syncwarp();
                next_chunk<COLS>(p, t, j, trow, tcol, st.base, lane);
            }
        }
    }

    // The copies of chunk j + AHEAD, or an empty group past the last, which keeps the groups counted.
    template <int COLS>
    static __device__ __forceinline__ void next_chunk(const Params& p, const Tile& t, int j, int trow, int tcol,
                                                      uint8_t* stage, int lane)
    {
        if (j + AHEAD < COLS / kChunk)
        {
            load_chunk(p, t, j + AHEAD, trow, tcol, stage, lane);
        }
        else
        {
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }

    static __device__ __forceinline__ float update(const Params& p, float w, float o)
    {
        w = __fsub_rn(w, __fmul_rn(p.decay, w));
        return __fsub_rn(w, __fmul_rn(p.step, o));
    }
    static __device__ __forceinline__ void pack_bf16(const float (&v)[kChunk], uint32_t (&w)[16])
    {
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
    }

    // The last product's result: written out, or applied to the weights, through the staging where TMA
    // can describe the destination, else element by element.
    static __device__ __forceinline__ void finish(const Params& p, const Tile& t, int trow, int col, uint8_t* in,
                                                  uint8_t* out, uint8_t* stage, int lane, float (&v)[kChunk])
    {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) v[i] *= 1.0f / kUnit;
        if (!p.vec)
        {
            finish_direct(p, t, trow + lane, col, v);
            return;
        }
        uint32_t w16[16];
        if constexpr (KIND == kMuon)
        {
            uint8_t* tile = SPLIT ? in : stage + 2 * kUnitBytes;
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                const float4 w = *reinterpret_cast<const float4*>(tile + tc::sw128_offset(lane, k));
                v[4 * k] = update(p, w.x, v[4 * k]);
                v[4 * k + 1] = update(p, w.y, v[4 * k + 1]);
                v[4 * k + 2] = update(p, w.z, v[4 * k + 2]);
                v[4 * k + 3] = update(p, w.w, v[4 * k + 3]);
            }
            put_f32(tile, lane, v);
            if constexpr (!SPLIT)
            {
                pack_bf16(v, w16);
                put_tile(out, lane, w16);
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0)
            {
                tc::tma_store_3d(&p.out, tile, col, trow, t.b);
                if constexpr (!SPLIT) tc::tma_store_3d(&p.out_t, out, col, trow, t.b);
                tc::bulk_commit_group();
            }
        }
        else
        {
            if constexpr (SPLIT)
            {
                put_f32(out, lane, v);
            }
            else
            {
                pack_bf16(v, w16);
                put_tile(out, lane, w16);
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0)
            {
                tc::tma_store_3d(&p.out, out, col, trow, t.b);
                tc::bulk_commit_group();
            }
        }
    }

    static __device__ __forceinline__ void finish_direct(const Params& p, const Tile& t, int row, int col,
                                                         float (&v)[kChunk])
    {
        if (row >= p.nrows)
        {
            return;
        }
        const int64_t at = p.stride_o * t.b + static_cast<int64_t>(row) * p.ldo + col;
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
        {
            if (col + i < p.ncols)
            {
                if constexpr (KIND == kMuon)
                {
                    float* w = static_cast<float*>(p.dst) + at + i;
                    *w = update(p, *w, v[i]);
                    if (p.lowp != nullptr) p.lowp[at + i] = __float2bfloat16_rn(*w);
                }
                else if (p.out_f32)
                {
                    static_cast<float*>(p.dst)[at + i] = v[i];
                }
                else
                {
                    static_cast<bf16*>(p.dst)[at + i] = __float2bfloat16_rn(v[i]);
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

template <int KIND, bool SPLIT>
int product(const char* what, const Params& p, cudaStream_t stream)
{
    const int clusters = pair::clusters_available<Work<KIND, SPLIT>, 8, SPLIT>();
    if (clusters < 1)
    {
        return fail(VEDA_ERR_UNSUPPORTED, std::string(what) + ": no CTA pair fits on this device");
    }
    return pair::launch_pair<Work<KIND, SPLIT>, 8, SPLIT>(what, p, std::min(p.total, clusters), stream);
}

// norm, X, then the products of every step; p's destination says what the last one (LAST) writes.
template <typename T, bool SPLIT, int LAST>
int iterate(const char* what, const Source& src, int64_t batch, int64_t rows, int64_t cols, int steps, float a,
            float b, float c, float eps, char* ws, Params p, cudaStream_t stream)
{
    const Layout l = layout(batch, rows, cols, SPLIT);
    double* partials = reinterpret_cast<double*>(ws + l.partials);
    uint16_t* x[2] = {reinterpret_cast<uint16_t*>(ws + l.x[0]), reinterpret_cast<uint16_t*>(ws + l.x[1])};
    uint16_t* sm[2] = {reinterpret_cast<uint16_t*>(ws + l.s), reinterpret_cast<uint16_t*>(ws + l.p)};
    const bool tall = rows > cols;
    const int64_t m = l.m, sp = l.planes * batch;
    // X of either buffer as S's operands, as M's partner (K-major boxes are 128 high) and written; S and
    // M read (they are symmetric: K-major always), written, and written transposed
    CUtensorMap xg[2], xa[2], xs[2], ml[2], ms[2], mt[2], dst{}, dst_low{};
    bool ok = true;
    for (int k = 0; k < 2; ++k)
    {
        ok = ok &&
             pair::make_map3(&xg[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 64, tall ? 64 : 128) &&
             pair::make_map3(&xa[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 64, tall ? 128 : 64) &&
             pair::make_map3(&xs[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 32, 32,
                             pair::Swizzle::k64) &&
             pair::make_map3(&ml[k], sm[k], 2, false, m, m, sp, l.lds, l.plane_s, 64, 128) &&
             pair::make_map3(&ms[k], sm[k], 2, false, m, m, sp, l.lds, l.plane_s, 32, 32, pair::Swizzle::k64) &&
             pair::make_map3(&mt[k], sm[k], 2, false, m, m, sp, l.lds, l.plane_s, 32, 32, pair::Swizzle::kNone);
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
    const bool f32 = LAST == kMuon || SPLIT;
    p.out_f32 = f32;
    p.vec = fits(p.dst, f32 ? 4 : 2) && (p.lowp == nullptr || fits(p.lowp, 2)) &&
            pair::make_map3(&dst, p.dst, f32 ? 4 : 2, !f32, cols, rows, batch, p.ldo, stride, 32, 32,
                            f32 ? pair::Swizzle::k128 : pair::Swizzle::k64) &&
            (p.lowp == nullptr || pair::make_map3(&dst_low, p.lowp, 2, true, cols, rows, batch, p.ldo, stride, 32, 32,
                                                  pair::Swizzle::k64));
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
    const int64_t tm = (m + 255) / 256, tr = (rows + 255) / 256, tc = (cols + 255) / 256;
    const int64_t half = tm * (tm + 1) / 2 * batch, whole = tr * tc * batch;
    if (half >= (1ll << 30) || whole >= (1ll << 30))
    {
        return fail(VEDA_ERR_INVALID_ARGUMENT, std::string(what) + ": too many tiles");
    }
    p.tall = tall;
    p.rows = static_cast<int>(rows);
    p.cols = static_cast<int>(cols);
    p.ca = a;
    p.cb = b;
    p.cc = c;
    p.tm = static_cast<int>(tm);
    p.by_n = pair::Divisor(static_cast<uint32_t>(tc));
    p.status = device_status_ptr();
    const pair::Divisor per_half(static_cast<uint32_t>(tm * (tm + 1) / 2)), per_whole(static_cast<uint32_t>(tr * tc));
    for (int k = 0; k < steps; ++k)
    {
        p.total = static_cast<int>(half);
        p.per_matrix = per_half;
        p.nrows = p.ncols = static_cast<int>(m);
        // S
        p.a = p.b = xg[k & 1];
        p.planes_a = p.planes_b = 2;
        p.k = static_cast<int>(std::max(rows, cols));
        p.out = ms[0];
        p.out_t = mt[0];
        rc = product<kGram, SPLIT>(what, p, stream);
        if (rc != VEDA_OK) return rc;
        // M
        p.a = p.b = ml[0];
        p.planes_a = p.planes_b = l.planes;
        p.k = static_cast<int>(m);
        p.src = sm[0];
        p.ld = l.lds;
        p.plane = l.plane_s;
        p.out = ms[1];
        p.out_t = mt[1];
        rc = product<kPoly, SPLIT>(what, p, stream);
        if (rc != VEDA_OK) return rc;
        // M X, or X M
        p.total = static_cast<int>(whole);
        p.per_matrix = per_whole;
        p.nrows = p.rows;
        p.ncols = p.cols;
        p.a = tall ? xa[k & 1] : ml[1];
        p.b = tall ? ml[1] : xa[k & 1];
        p.planes_a = tall ? 2 : l.planes;
        p.planes_b = tall ? l.planes : 2;
        p.src = x[k & 1];
        p.ld = l.ldx;
        p.plane = l.plane_x;
        p.out = k < steps - 1 ? xs[(k + 1) & 1] : dst;
        p.out_t = dst_low;
        rc = k < steps - 1 ? product<kApply, SPLIT>(what, p, stream) : product<LAST, SPLIT>(what, p, stream);
        if (rc != VEDA_OK) return rc;
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
    const ns::Source src{g, ldg, stride_g, nullptr, 0.0f, 0, nullptr, 1.0f, 1.0f, 0};
    char* ws = static_cast<char*>(workspace);
    return split ? ns::iterate<float, true, ns::kOut>("veda_orthogonalize", src, batch, rows, cols, steps, a, b, c, eps,
                                                      ws, p, stream)
                 : ns::iterate<bf16, false, ns::kOut>("veda_orthogonalize", src, batch, rows, cols, steps, a, b, c, eps,
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
    p.dst = master;
    p.lowp = static_cast<bf16*>(lowp);
    p.ldo = cols;
    p.stride_o = stride;
    p.decay = lr * weight_decay;
    p.step = lr * update_scale;
    p.sumsq = sumsq;
    p.grad_scale = grad_scale;
    p.flags = flags;
    const ns::Source src{grad, cols, stride, momentum, beta, nesterov, sumsq, max_norm, grad_scale, flags};
    char* ws = static_cast<char*>(workspace);
    return split ? ns::iterate<float, true, ns::kMuon>("veda_muon_step", src, batch, rows, cols, steps, a, b, c, eps, ws,
                                                       p, stream)
                 : ns::iterate<float, false, ns::kMuon>("veda_muon_step", src, batch, rows, cols, steps, a, b, c, eps, ws,
                                                        p, stream);
}
