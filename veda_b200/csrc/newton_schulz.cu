// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step built on it.
//
// For each matrix of a batch, X = G / (|G|_F + eps), then `steps` times
//   S = X X^T (of the smaller side),  M = a I + b S + c S^2,  X <- M X,
// the odd quintic a s + b s^3 + c s^5 applied to every singular value. All 3 x steps products of all
// matrices are one launch of the persistent CTA-pair tensor-core kernel (pair_mma.cuh): the tiles are
// listed step by step, matrix by matrix, and a tile of a step starts once every tile of the same
// matrix's step before it is stored, which a counter per matrix and step tells. With a few matrices the
// next step of one runs beside the last tiles of another, so neither the last, partly filled wave of a
// product nor its epilogue leaves SMs idle. As one launch per product, 28 x 1024 x 1024 took 870 us
// against 760, both in short runs at full clocks (long ones, under the power cap: 850). A tall matrix is multiplied from the other side (S = X^T X, X <- X M) by operand
// order alone, so nothing is transposed. S and M are symmetric: the tiles on and above the diagonal are
// computed, and each one above it is written a second time, transposed.
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
#include <atomic>
#include <type_traits>

namespace veda::cuda
{
int* device_status_ptr();

namespace ns
{

constexpr float kUnit = 1024.0f;   // stored value = kUnit x value

// What a tile computes: S, M, the next X, or the last X as a result or as the weights' update.
enum Kind { kGram, kPoly, kApply, kOut, kMuon };

struct Params
{
    // X of either buffer as S's operands and as M's partner, S and M: planes hi, lo of each matrix
    // (K-major boxes of 64 x 128, MN-major ones of 64 x 64)
    CUtensorMap xg[2], xa[2], s, m;
    // what is written, in boxes of 32 x 32: X of either buffer, S and M as they are and transposed, the
    // destination (kMuon: fp32 weights) and the bf16 weights
    CUtensorMap x_out[2], s_out, s_out_t, m_out, m_out_t, dst_out, lowp_out;
    int tall;
    int rows, cols;          // of X
    int side;                // of S and M: the smaller of them
    int planes;              // of S and M
    int batch, steps;
    int tn, half, whole;     // column tiles of S; tiles of S or M of one matrix, of X of one matrix
    int sym_tiles, iteration;   // tiles of S of all matrices; of an iteration
    pair::Divisor by_iteration, by_sym, by_half, by_whole, by_n;
    float ca, cb, cc;
    const uint16_t *x[2], *s_ptr;   // read by the epilogues
    int64_t ldx, plane_x, lds, plane_s;
    unsigned* counters;      // [batch][3 steps] finished epilogue warps
    // kOut, kMuon: the destination, stored by TMA if vec
    void* dst;
    int64_t ldo, stride_o;
    int out_f32, vec;
    bf16* lowp;
    float decay, step;       // lr weight_decay, lr scale
    const double* sumsq;
    float grad_scale;
    int flags;
    int* status;
};

struct Tile
{
    bool skip, a_mn, b_mn;
    int kbs, b, mb, nb, kind, k;
    uint32_t idesc;
};

// What a kind of tile reads and writes in its epilogue.
struct View
{
    const CUtensorMap *out, *out_t;
    int nrows, ncols;
    const uint16_t* src;     // kPoly: S; later kinds: X
    int64_t ld, plane;
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

template <int KIND, bool SPLIT, int TN>
struct Part
{
    static constexpr bool SYM = KIND <= kPoly;

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
    static __device__ __forceinline__ void copy_plane(uint8_t* tile, const uint16_t* src, const View& w, int row,
                                                      int col, int lane)
    {
        const int seg = lane & 3, c = col + seg * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const int r = 8 * k + (lane >> 2);
            const bool in = row + r < w.nrows && c < w.ncols;
            copy16(tile + swz64(r, seg), in ? src + (row + r) * w.ld + c : src, in);
        }
    }

    // Starts the copies of chunk j, one group (empty where nothing is read).
    static __device__ __forceinline__ void load_chunk(const Params& p, const View& w, const Tile& t, int j, int trow, int tcol,
                                                      uint8_t* stage, int lane)
    {
        uint8_t* in = stage + in_unit(j) * kUnitBytes;
        const int col = tcol + j * kChunk;
        if constexpr (KIND == kPoly)
        {
            const uint16_t* src = w.src + w.plane * p.planes * t.b;
            copy_plane(in, src, w, trow, col, lane);
            if constexpr (SPLIT) copy_plane(in + kUnitBytes, src + w.plane, w, trow, col, lane);
        }
        if constexpr (READS_X)
        {
            copy_plane(in, w.src + w.plane * (2 * t.b + 1), w, trow, col, lane);
        }
        if constexpr (KIND == kMuon)
        {
            if (p.vec)
            {
                uint8_t* tile = SPLIT ? in : stage + 2 * kUnitBytes;
                const float* weights = static_cast<const float*>(p.dst) + p.stride_o * t.b;
                const int seg = lane & 7, c = col + seg * 4;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    const int r = 4 * k + (lane >> 3);
                    const bool inside = trow + r < w.nrows && c < w.ncols;
                    copy16(tile + tc::sw128_offset(r, seg), inside ? weights + (trow + r) * p.ldo + c : weights, inside);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    static __device__ __forceinline__ void before(const Params& p, const View& w, const Tile& t, int row0, int col0,
                                                  uint8_t* stage, int lane)
    {
        if constexpr (AHEAD > 0)
        {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
            {
                load_chunk(p, w, t, j, t.mb * pair::kTile + row0, t.nb * TN + col0, stage, lane);
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
    static __device__ __forceinline__ void epilogue(const Params& p, const View& w, const Tile& t, uint32_t taddr,
                                                    int row0, int col0, uint8_t* stage, int lane)
    {
        const int trow = t.mb * pair::kTile + row0, tcol = t.nb * TN + col0;
        if (trow >= w.nrows || (KIND == kMuon && skipped_step(p.flags, p.sumsq, p.grad_scale)))
        {
            landed();
            return;
        }
        const bool mirror = SYM && t.nb >= (pair::kTile / TN) * (t.mb + 1);   // right of the diagonal tiles
        // the tile's sums carry kUnit^2; what is stored carries kUnit
        const float f = (KIND == kPoly ? p.cc : 1.0f) / kUnit;
#pragma unroll 1
        for (int j = 0; j < COLS / kChunk; ++j)
        {
            const int col = tcol + j * kChunk;
            if (col >= w.ncols)
            {
                break;
            }
            uint8_t* in = stage + in_unit(j) * kUnitBytes;
            uint8_t* out = stage + out_unit(j) * kUnitBytes;
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
                    next_chunk<COLS>(p, w, t, j, trow, tcol, stage, lane);
                }
                if (lane == 0)
                {
                    tc::bulk_wait_group_read<OUTS - 1>();   // the stores that last used `out` have read it
                }
                __syncwarp();
            }
            if constexpr (KIND == kOut || KIND == kMuon)
            {
                finish(p, w, t, trow, col, in, out, stage, lane, v);
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
                    tc::tma_store_3d(w.out, out, col, trow, z);
                    if constexpr (PLANES == 2) tc::tma_store_3d(w.out, out + kUnitBytes, col, trow, z + 1);
                    if (mirror)
                    {
                        tc::tma_store_3d(w.out_t, out + PLANES * kUnitBytes, trow, col, z);
                        if constexpr (PLANES == 2) tc::tma_store_3d(w.out_t, out + 3 * kUnitBytes, trow, col, z + 1);
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
                next_chunk<COLS>(p, w, t, j, trow, tcol, stage, lane);
            }
        }
        landed();
    }

    // Chunks of rows or columns past the end are copied in (as zeros) and not used: they have landed before
    // the warp leaves the tile, since the next one's kind may write to their units without copies of its own
    // to wait for.
    static __device__ __forceinline__ void landed()
    {
        if constexpr (AHEAD > 0)
        {
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
        }
    }

    // The copies of chunk j + AHEAD, or an empty group past the last, which keeps the groups counted.
    template <int COLS>
    static __device__ __forceinline__ void next_chunk(const Params& p, const View& w, const Tile& t, int j, int trow, int tcol,
                                                      uint8_t* stage, int lane)
    {
        if (j + AHEAD < COLS / kChunk)
        {
            load_chunk(p, w, t, j + AHEAD, trow, tcol, stage, lane);
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
    // can describe the destination, else by rows of 32 elements.
    static __device__ __forceinline__ void finish(const Params& p, const View& w, const Tile& t, int trow, int col, uint8_t* in,
                                                  uint8_t* out, uint8_t* stage, int lane, float (&v)[kChunk])
    {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) v[i] *= 1.0f / kUnit;
        if (!p.vec)
        {
            // two units, 4 KB: a set of the split forms, else units 2 and 3, which only stores use that are
            // not made here
            uint8_t* tile = !SPLIT ? stage + 2 * kUnitBytes : KIND == kMuon ? in : out;
            put_f32(tile, lane, v);
            __syncwarp();
            finish_direct(p, w, t, trow, col + lane, tile, lane);
            __syncwarp();
            if (lane == 0) tc::bulk_commit_group();   // empty: the waits above count groups
            return;
        }
        uint32_t w16[16];
        if constexpr (KIND == kMuon)
        {
            uint8_t* tile = SPLIT ? in : stage + 2 * kUnitBytes;
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                const float4 old = *reinterpret_cast<const float4*>(tile + tc::sw128_offset(lane, k));
                v[4 * k] = update(p, old.x, v[4 * k]);
                v[4 * k + 1] = update(p, old.y, v[4 * k + 1]);
                v[4 * k + 2] = update(p, old.z, v[4 * k + 2]);
                v[4 * k + 3] = update(p, old.w, v[4 * k + 3]);
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
                tc::tma_store_3d(w.out, tile, col, trow, t.b);
                if constexpr (!SPLIT) tc::tma_store_3d(w.out_t, out, col, trow, t.b);
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
                tc::tma_store_3d(w.out, out, col, trow, t.b);
                tc::bulk_commit_group();
            }
        }
    }

    // The staged chunk row by row, a column a lane: whole lines of rows that start anywhere. With a row a
    // lane, each store to 32 lines, Muon on 3 x 1111 x 2222 took 670 us instead of 495.
    static __device__ __forceinline__ void finish_direct(const Params& p, const View& w, const Tile& t, int trow, int col,
                                                         const uint8_t* tile, int lane)
    {
        if (col >= w.ncols)
        {
            return;
        }
        const int n = min(32, w.nrows - trow);
        const int64_t at = p.stride_o * t.b + static_cast<int64_t>(trow) * p.ldo + col;
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 8)
        {
            float old[8];
            if constexpr (KIND == kMuon)
            {
#pragma unroll
                for (int i = 0; i < 8; ++i) old[i] = i0 + i < n ? static_cast<const float*>(p.dst)[at + (i0 + i) * p.ldo] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const int r = i0 + i;
                if (r < n)
                {
                    const int64_t here = at + r * p.ldo;
                    const float v = *reinterpret_cast<const float*>(tile + tc::sw128_offset(r, lane >> 2) + (lane & 3) * 4);
                    if constexpr (KIND == kMuon)
                    {
                        const float x = update(p, old[i], v);
                        static_cast<float*>(p.dst)[here] = x;
                        if (p.lowp != nullptr) p.lowp[here] = __float2bfloat16_rn(x);
                    }
                    else if (p.out_f32)
                    {
                        static_cast<float*>(p.dst)[here] = v;
                    }
                    else
                    {
                        static_cast<bf16*>(p.dst)[here] = __float2bfloat16_rn(v);
                    }
                }
            }
        }
    }
};

// The tiles of all products, step by step and matrix by matrix. LAST: kOut or kMuon.
template <int LAST, bool SPLIT, int TN_>
struct Work
{
    static constexpr int TN = TN_;
    // The iteration amplifies what a chain's truncation takes off (7 times at 256 x 6000): 1.2e-5 of the result with
    // chains of 4, 6.4e-6 with 2, 3.9e-6 with 1, for 1001 x 523 in 216, 234 and 311 us.
    static constexpr int CHAIN = 2;
    using Params = ns::Params;
    using Tile = ns::Tile;
    struct State
    {
    };
    static constexpr unsigned kArrivals = 16;   // epilogue warps of a CTA pair

    static __device__ __forceinline__ bool tile(const Params& p, int cid, int clusters, int i, Tile& t)
    {
        int r;
        t.k = p.by_iteration.div(cid + i * clusters, r);
        if (t.k >= p.steps)
        {
            return false;
        }
        if (r < 2 * p.sym_tiles)
        {
            t.kind = p.by_sym.div(r, r);   // kGram, kPoly
            t.b = p.by_half.div(r, r);
            // row mb of the upper triangle holds the tiles from column tile mb kTile / TN on
            t.mb = 0;
            t.nb = 0;
            while (r >= p.tn - t.nb)
            {
                r -= p.tn - t.nb;
                ++t.mb;
                t.nb += pair::kTile / TN;
            }
            t.nb += r;
        }
        else
        {
            t.kind = kApply;
            t.b = p.by_whole.div(r - 2 * p.sym_tiles, r);
            t.mb = p.by_n.div(r, t.nb);
        }
        t.skip = false;
        const int terms = t.kind == kGram ? (p.tall ? p.rows : p.cols) : p.side;
        t.kbs = (terms + pair::kBK - 1) / pair::kBK;
        // tall: S = X^T X, X M; else S = X X^T, M X; S and M read as they are, being symmetric
        t.a_mn = t.kind == kGram && p.tall;
        t.b_mn = t.kind == kGram ? p.tall != 0 : t.kind != kPoly && p.tall == 0;
        t.idesc = pair::idesc<TN>(false, t.a_mn, t.b_mn);
        return true;
    }

    static __device__ __forceinline__ void operands(const Params& p, const Tile& t, int rank, pair::Piece& a,
                                                    pair::Piece& b)
    {
        const int m = t.mb * pair::kTile + rank * 128, n = t.nb * TN + rank * (TN / 2);
        const CUtensorMap* x = t.kind == kGram ? &p.xg[t.k & 1] : &p.xa[t.k & 1];
        const bool x_first = t.kind == kGram || (t.kind == kApply && p.tall);
        const bool x_second = t.kind == kGram || (t.kind == kApply && !p.tall);
        const CUtensorMap* sym = t.kind == kPoly ? &p.s : &p.m;
        a = {x_first ? x : sym, t.a_mn ? m : 0, t.a_mn ? 0 : m, (x_first ? 2 : p.planes) * t.b};
        b = {x_second ? x : sym, t.b_mn ? n : 0, t.b_mn ? 0 : n, (x_second ? 2 : p.planes) * t.b};
    }
    static __device__ __forceinline__ void prefetch(const Params& p)
    {
        tc::tma_prefetch(&p.xg[0]);
        tc::tma_prefetch(&p.s);
        tc::tma_prefetch(&p.m);
        tc::tma_prefetch(&p.xa[0]);
    }

    // Waits (bounded) until the matrix's step before is stored: its counter is full.
    static __device__ __forceinline__ void ready(const Params& p, const Tile& t, volatile int* abort)
    {
        const int step = 3 * t.k + t.kind;
        if (step == 0)
        {
            return;
        }
        const unsigned want = kArrivals * static_cast<unsigned>(t.kind == kGram ? p.whole : p.half);
        const unsigned* c = p.counters + static_cast<int64_t>(t.b) * 3 * p.steps + step - 1;
        const auto full = [&] {
            unsigned have;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(have) : "l"(c) : "memory");
            return have >= want;
        };
        if (!full())
        {
            const long long start = clock64();
            while (!full())
            {
                if (*abort != 0)
                {
                    break;
                }
                if (clock64() - start > tc::kWaitBudget)
                {
                    *abort = 1;
                    if (p.status != nullptr) atomicExch(p.status, VEDA_ERR_TIMEOUT);
                    break;
                }
            }
        }
        // what other SMs stored is read by TMA next
        asm volatile("fence.proxy.async.global;" ::: "memory");
    }

    static __device__ __forceinline__ View view(const Params& p, const Tile& t)
    {
        View w;
        if (t.kind == kGram)
        {
            w = {&p.s_out, &p.s_out_t, p.side, p.side, nullptr, 0, 0};
        }
        else if (t.kind == kPoly)
        {
            w = {&p.m_out, &p.m_out_t, p.side, p.side, p.s_ptr, p.lds, p.plane_s};
        }
        else
        {
            const bool last = t.k == p.steps - 1;
            w = {last ? &p.dst_out : &p.x_out[(t.k + 1) & 1], &p.lowp_out, p.rows, p.cols, p.x[t.k & 1], p.ldx, p.plane_x};
        }
        return w;
    }

    // A function of the Part that the tile's kind names.
    template <typename F>
    static __device__ __forceinline__ void with_part(const Params& p, const Tile& t, F&& f)
    {
        if (t.kind == kGram) f(Part<kGram, SPLIT, TN>{});
        else if (t.kind == kPoly) f(Part<kPoly, SPLIT, TN>{});
        else if (t.k < p.steps - 1) f(Part<kApply, SPLIT, TN>{});
        else f(Part<LAST, SPLIT, TN>{});
    }

    static __device__ __forceinline__ void before(const Params& p, const Tile& t, State&, int row0, int col0,
                                                  pair::Staging& st, int lane, volatile int* abort)
    {
        if (t.kind == kGram)
        {
            return;   // its epilogue reads nothing
        }
        if (lane == 0)
        {
            ready(p, t, abort);
        }
        __syncwarp();
        const View w = view(p, t);
        with_part(p, t, [&](auto part) { part.before(p, w, t, row0, col0, st.base, lane); });
    }

    template <int COLS>
    static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, State&, uint32_t taddr,
                                                    int row0, int col0, pair::Staging& st, int lane)
    {
        const View w = view(p, t);
        with_part(p, t, [&](auto part) { part.template epilogue<COLS>(p, w, t, taddr, row0, col0, st.base, lane); });
    }

    // The warp's share of the tile is stored: counts it.
    static __device__ __forceinline__ void after(const Params& p, const Tile& t, int lane)
    {
        if (lane == 0)
        {
            tc::bulk_wait_group<0>();
            asm volatile("fence.proxy.async.global;" ::: "memory");
            unsigned* c = p.counters + static_cast<int64_t>(t.b) * 3 * p.steps + 3 * t.k + t.kind;
            asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(c) : "memory");
        }
        __syncwarp();
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

// What X's stored values are made with: kUnit u / (|u| + eps) = (u lift) scale, from the sum of squares. lift is a
// power of two that keeps scale a normal number for norms below 2^-100 and above 2^100 (a scale of 2^10 / |u| in fp32
// would be infinite below 2^-118). 0 where norm and eps both are: such a matrix is zero and stays so.
struct Unit
{
    float lift, scale;
    __device__ __forceinline__ float operator()(float u) const { return u * lift * scale; }
};
__device__ __forceinline__ Unit unit_of(double sum, float eps)
{
    const double d = sqrt(sum) + static_cast<double>(eps);
    const double lift = d < 0x1p-100 ? 0x1p64 : d > 0x1p100 ? 0x1p-64 : 1.0;
    return {static_cast<float>(lift), d == 0.0 ? 0.0f : static_cast<float>(static_cast<double>(kUnit) / (d * lift))};
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

// X's two planes: 1024 u / (|u| + eps), the norm summed from the blocks' partials in a fixed order; and
// the matrix's counters, cleared.
template <typename T, int N>
__global__ void __launch_bounds__(256)
init_kernel(Source s, int rows, int cols, const double* __restrict__ partials, float eps, uint16_t* __restrict__ x,
            int64_t ldx, int64_t plane, unsigned* __restrict__ counters, int steps)
{
    __shared__ double part[8];
    dep_wait();
    dep_release();
    if (blockIdx.x == 0)
    {
        for (int i = threadIdx.x; i < 3 * steps; i += 256) counters[static_cast<int64_t>(blockIdx.y) * 3 * steps + i] = 0;
    }
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
    const Unit unit = unit_of(total, eps);
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
                const float v = unit(u[k]);
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

// ---- small matrices: the whole iteration in one block ------------------------------------------
// A matrix whose smaller side is at most 128 and whose larger side is at most 256 stays in one SM from
// its norm to the result: X, then S and M in turn, as hi and lo planes in shared memory (128-byte
// swizzle, blocks of 128 rows x 64 columns), S, S^2 and M X in tensor memory, 16 warps between them.
// X is held with its smaller side as rows, a tall matrix transposed on the way in and out. The block
// of columns that is K-major for S = X X^T is MN-major for M X without moving a byte. Products are split
// (hi lo + lo hi + hi hi) for either dtype: what such a matrix costs is the latency of its 15 products
// one after the other, not their size. As 17 launches of the tiled kernels the two 192 x 64 matrices
// took 81 us on the GPU; in one block each, 28.7 us. At this size fetching instructions that run once costs
// as much as what they do: passes that stop where the whole block has nothing left, one copy of each, and shifts
// for divisions took the fp32 Muon step of 2 x 64 x 64 from 24.7 to 19 us.
// CLUSTER: a longer side of up to 4096 is cut among the up to 16 blocks of a cluster. Each multiplies its
// columns of X; only S needs them all, and its parts meet in the blocks' shared memory: every block adds
// some rows and hands their sums to the others. M, one product of the small side, is formed by each. An
// iteration then takes 8 (64 x 4096) to 15 us (128 x 4096, 16 blocks), 3 to 7 of them for the exchange;
// 128 x 1024 in fp32 went from 142 us (tiled) to 75, 64 x 4096 from 277 to 49.
struct Small
{
    Source src;
    int rows, cols, steps;
    float ca, cb, cc, eps;
    void* dst;               // result, or the fp32 weights
    int64_t ldo, stride_o;
    bf16* lowp;
    float decay, step;
    int vec, vec_out;        // source rows can be read, result rows written, four elements at a time
    int* status;
    // how the longer side is cut: blocks of a matrix, columns each (the last may have fewer), rows of S
    // that each adds up, bytes for S
    int ranks, share, band, s_bytes;
    // log2 of the items that a row (in; tall: a quarter of it) and a result's row (out) take in a block's count:
    // padded to powers of two, since dividing costs more than the idle turns
    int in_log, out_log, s_log;
};

constexpr int kMaxRanks = 16;
constexpr int kSmallSide = 128, kSmallLong = 256;
constexpr int kSmallThreads = 512;
constexpr int kBlockBytes = 128 * 128;   // 128 rows of 64 fp16

// Fills in the cut; the shared memory of a block.
inline int small_smem(Small& p)
{
    const int m = std::min(p.rows, p.cols), n = std::max(p.rows, p.cols), m16 = (m + 15) / 16 * 16;
    p.ranks = (n + kSmallLong - 1) / kSmallLong;
    p.share = ((n + p.ranks - 1) / p.ranks + 15) / 16 * 16;
    p.band = (m16 + p.ranks - 1) / p.ranks;
    const auto log_of = [](int items) {
        int k = 0;
        while ((1 << k) < items) ++k;
        return k;
    };
    const int own_cols = p.rows > p.cols ? p.cols : p.ranks > 1 ? p.share : p.cols;
    const int in = p.vec ? own_cols / 4 : own_cols;
    p.in_log = log_of(p.rows > p.cols ? (in + 3) / 4 : in);
    p.out_log = log_of(p.vec_out ? own_cols / 4 : own_cols);
    p.s_log = log_of(m16 / 4);
    p.s_bytes = std::max(2 * ((m + 63) / 64) * kBlockBytes, p.ranks > 1 ? m16 * (m16 + 4) * 4 : 0);
    return 2 * ((p.share + 63) / 64) * kBlockBytes + p.s_bytes + 1024 + 256;
}

// Byte offset of element (row, col) of a plane.
__device__ __forceinline__ uint32_t plane_at(int row, int col)
{
    return static_cast<uint32_t>((col >> 6) * kBlockBytes) + tc::sw128_offset(row, (col & 63) >> 3) + (col & 7) * 2;
}

__device__ __forceinline__ void store_four(float* p, const float (&v)[4])
{
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_four(bf16* p, const float (&v)[4])
{
    alignas(8) __nv_bfloat162 b[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(b);
}

// 32 columns from `col` of the lane's row as hi and lo: 1024 x value = v.
__device__ __forceinline__ void put_planes(uint8_t* hi, uint8_t* lo, int row, int col, const float (&v)[32])
{
    const uint32_t block = static_cast<uint32_t>((col >> 6) * kBlockBytes);
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float x = v[8 * k + 2 * i], y = v[8 * k + 2 * i + 1];
            h[i] = pack_f16(x, y);
            const float2 back = unpack_f16(h[i]);
            l[i] = pack_f16(x - back.x, y - back.y);
        }
        const uint32_t at = block + tc::sw128_offset(row, ((col & 63) >> 3) + k);
        *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
    }
}

template <typename T, bool MUON, bool CLUSTER>
__global__ void __launch_bounds__(kSmallThreads, 1)
small_kernel(const Small p)
{
    using namespace tc;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const bool tall = p.rows > p.cols;
    // this block's matrix, and its part of the longer side: n columns from `from` on
    const int ranks = CLUSTER ? p.ranks : 1;
    const int rank = CLUSTER ? static_cast<int>(pair::cluster_rank()) : 0;
    const int matrix = static_cast<int>(blockIdx.x) / ranks;
    const int m = tall ? p.cols : p.rows, from = rank * p.share;
    const int n = min((tall ? p.rows : p.cols) - from, p.share);
    const int own_rows = tall ? n : p.rows, own_cols = tall ? p.cols : n;
    const int m16 = (m + 15) & ~15, n16 = (n + 15) & ~15;
    const int nb = (p.share + 63) >> 6, sb = (m + 63) >> 6;   // the same layout in every block of a cluster
    uint8_t* const xh = smem;
    uint8_t* const xl = xh + nb * kBlockBytes;
    uint8_t* const sh = xl + nb * kBlockBytes;
    uint8_t* const sl = sh + sb * kBlockBytes;
    uint64_t* const done = reinterpret_cast<uint64_t*>(sh + p.s_bytes);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* const abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    __shared__ double part[kSmallThreads / 32];
    __shared__ Unit shared_unit;
    __shared__ double shares[kMaxRanks];
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0)
    {
        *abort = 0;
        mbar_init(done, 1);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    if ((m | n) & 15)
    {
        // what pads the products' 16-term steps is zero
        for (int i = threadIdx.x; i < 2 * nb * kBlockBytes / 16; i += kSmallThreads)
        {
            reinterpret_cast<uint4*>(xh)[i] = make_uint4(0, 0, 0, 0);
        }
    }
    fence_before();
    __syncthreads();
    if constexpr (CLUSTER) pair::cluster_sync();   // every block runs: its shared memory may be written
    fence_after();
    const uint32_t tmem = *tmem_slot;
    dep_wait();
    dep_release();

    const bool skip = skipped_step(p.src.flags, p.src.sumsq, p.src.grad_scale);
    if (!skip)
    {
        // the norm (and the momentum), then X
        const Source& s = p.src;
        const float clip = clip_scale(s.sumsq, s.max_norm, s.grad_scale);
        const int64_t first = s.stride * matrix + (tall ? from * s.ld : from);
        const T* g = static_cast<const T*>(s.g) + first;
        float* mom = MUON ? s.momentum + first : nullptr;
        const auto advance = [&](float& x, float& o) {
            x = seen(x, s.grad_scale, clip);
            o = fmaf(s.beta, o, x);
            x = s.nesterov ? fmaf(s.beta, o, x) : o;
        };
        // An item is four elements of a row where they can be read together, else one. A wide matrix's items go
        // to the threads along its rows; a tall one's in tiles of 8 rows x 4 items a warp, since a row of it
        // becomes a column here and lanes side by side would write to the same banks.
        const int step = p.vec ? 4 : 1, in_log = p.in_log;
        const auto place = [&](int e, int& r, int& c) {
            if (tall)
            {
                const int tile = e >> 5;
                r = (tile >> in_log) * 8 + ((e >> 2) & 7);
                c = ((tile & ((1 << in_log) - 1)) * 4 + (e & 3)) * step;
            }
            else
            {
                r = e >> in_log;
                c = (e & ((1 << in_log) - 1)) * step;
            }
            return r < own_rows && c < own_cols;
        };
        const auto store = [&](int r, int c, const float (&u)[4], const Unit& unit) {
            alignas(8) __half h[4], l[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                const float v = unit(u[k]);
                h[k] = __float2half_rn(v);
                l[k] = __float2half_rn(v - __half2float(h[k]));
            }
            if (!tall && p.vec)
            {
                const uint32_t at = plane_at(r, c);   // 8 bytes of a 16-byte group
                *reinterpret_cast<uint2*>(xh + at) = *reinterpret_cast<const uint2*>(h);
                *reinterpret_cast<uint2*>(xl + at) = *reinterpret_cast<const uint2*>(l);
                return;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                if (k < step)
                {
                    const uint32_t at = tall ? plane_at(c + k, r) : plane_at(r, c + k);
                    *reinterpret_cast<__half*>(xh + at) = h[k];
                    *reinterpret_cast<__half*>(xl + at) = l[k];
                }
            }
        };
        // Up to 32768 elements, 64 a thread: the last half (or all) stays in registers until the norm is known, what
        // comes before it waits in the place of S, 64 KB where there is a first half. All loads of a
        // round before the first store: Muon's momentum could alias what is read.
        constexpr int kItems = 8;
        const int count = tall ? ((own_rows + 7) / 8) << (in_log + 5) : own_rows << in_log;
        const int each = kItems * (p.vec ? 1 : 4) * kSmallThreads;   // items of a round
        float* const waiting = reinterpret_cast<float*>(sh);
        float u[kItems][4];
        double sum = 0.0;
        const auto round = [&](int base) {
#pragma unroll
            for (int q = 0; q < kItems; ++q)
            {
#pragma unroll
                for (int k = 0; k < 4; ++k) u[q][k] = 0.0f;
            }
            if (p.vec)
            {
                float o[MUON ? kItems : 1][4];
#pragma unroll
                for (int q = 0; q < kItems; ++q)
                {
                    int r, c;
                    const int e = base + static_cast<int>(threadIdx.x) + q * kSmallThreads;
                    if (base + q * kSmallThreads >= count) break;   // the whole block: what is not run is not fetched
                    if (e < count && place(e, r, c))
                    {
                        load_n<T, 4>(g + (r * s.ld + c), u[q]);
                        if constexpr (MUON) load_n<float, 4>(mom + (r * s.ld + c), o[q]);
                    }
                }
                if constexpr (MUON)
                {
#pragma unroll
                    for (int q = 0; q < kItems; ++q)
                    {
                        int r, c;
                        const int e = base + static_cast<int>(threadIdx.x) + q * kSmallThreads;
                        if (base + q * kSmallThreads >= count) break;
                        if (e < count && place(e, r, c))
                        {
#pragma unroll
                            for (int k = 0; k < 4; ++k) advance(u[q][k], o[q][k]);
                            *reinterpret_cast<float4*>(mom + (r * s.ld + c)) = make_float4(o[q][0], o[q][1], o[q][2], o[q][3]);
                        }
                    }
                }
            }
            else
            {
                float o[MUON ? kItems : 1][4];
#pragma unroll
                for (int q = 0; q < kItems * 4; ++q)
                {
                    int r, c;
                    const int e = base + static_cast<int>(threadIdx.x) + q * kSmallThreads;
                    const bool in = e < count && place(e, r, c);
                    u[q / 4][q % 4] = in ? to_f32(g[r * s.ld + c]) : 0.0f;
                    if constexpr (MUON) o[q / 4][q % 4] = in ? mom[r * s.ld + c] : 0.0f;
                }
                if constexpr (MUON)
                {
#pragma unroll
                    for (int q = 0; q < kItems * 4; ++q)
                    {
                        int r, c;
                        const int e = base + static_cast<int>(threadIdx.x) + q * kSmallThreads;
                        if (e < count && place(e, r, c))
                        {
                            advance(u[q / 4][q % 4], o[q / 4][q % 4]);
                            mom[r * s.ld + c] = o[q / 4][q % 4];
                        }
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < kItems; ++q)
            {
                if (base + q * kSmallThreads >= count) break;
#pragma unroll
                for (int k = 0; k < 4; ++k) sum += static_cast<double>(u[q][k]) * u[q][k];
            }
        };
        const auto planes = [&](int base, const Unit& unit) {
#pragma unroll
            for (int q = 0; q < kItems; ++q)
            {
                const int t = static_cast<int>(threadIdx.x);
                int r, c;
                if (p.vec)
                {
                    const int e = base + t + q * kSmallThreads;
                    if (base + q * kSmallThreads >= count) break;
                    if (e < count && place(e, r, c)) store(r, c, u[q], unit);
                    continue;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                {
                    const int e = base + t + (q * 4 + k) * kSmallThreads;
                    const float one[4] = {u[q][k], 0.0f, 0.0f, 0.0f};
                    if (base + (q * 4 + k) * kSmallThreads >= count) break;
                    if (e < count && place(e, r, c)) store(r, c, one, unit);
                }
            }
        };
        const bool twice = count > each;
#pragma unroll 1
        for (int base = 0; base < count; base += each)
        {
            round(base);
            if (base + each < count)
            {
#pragma unroll
                for (int q = 0; q < kItems; ++q)
                {
                    reinterpret_cast<float4*>(waiting)[q * kSmallThreads + threadIdx.x] = make_float4(u[q][0], u[q][1], u[q][2], u[q][3]);
                }
            }
        }
        sum = warp_sum(sum);
        if (lane == 0) part[warp] = sum;
        __syncthreads();
        if (warp == 0)
        {
            sum = warp_sum(lane < kSmallThreads / 32 ? part[lane] : 0.0);
            if constexpr (CLUSTER)
            {
                // every block gets every block's sum and adds them in rank order
                if (lane < ranks)
                {
                    const uint32_t to = pair::peer_addr(&shares[rank], lane);
                    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(sum) : "memory");
                }
                pair::cluster_arrive();
                pair::cluster_wait();
                sum = 0.0;
                for (int k = 0; k < ranks; ++k) sum += shares[k];
            }
            if (lane == 0)
            {
                shared_unit = unit_of(sum, p.eps);
            }
        }
        else if constexpr (CLUSTER)
        {
            pair::cluster_arrive();
            pair::cluster_wait();
        }
        __syncthreads();
        const Unit unit = shared_unit;
#pragma unroll 1
        for (int base = twice ? each : 0; base >= 0; base -= each)
        {
            planes(base, unit);
            if (base > 0)
            {
#pragma unroll
                for (int q = 0; q < kItems; ++q)
                {
                    const float4 w = reinterpret_cast<const float4*>(waiting)[q * kSmallThreads + threadIdx.x];
                    u[q][0] = w.x, u[q][1] = w.y, u[q][2] = w.z, u[q][3] = w.w;
                }
            }
        }
    }

    const uint32_t ts = tmem, tx = tmem + 128;   // S or S^2; M X
    const int quarter = warp & 3, half = warp >> 2;   // TMEM lanes, and which quarter of the columns
    const int row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    uint32_t phase = 0;
    // D = A B over `terms` (a multiple of 16) from the planes of a and b; thread 0 issues
    const auto product = [&](uint32_t d, const uint8_t* ah, const uint8_t* al, const uint8_t* bh, const uint8_t* bl,
                             auto b_mn, int cols_, int terms) {
        fence_proxy_async();
        fence_before();
        __syncthreads();
        if (warp == 0)
        {
            fence_after();
            // The whole warp works out the descriptors, in registers that it shares, and one lane issues:
            // under a branch for one thread each product took 100 to 130 cycles to issue.
            const bool leader = pair::elect_one();
            const uint32_t idesc = (1u << 4) | ((decltype(b_mn)::value ? 1u : 0u) << 16) |
                                   (static_cast<uint32_t>(cols_ >> 3) << 17) | (8u << 24);
            constexpr uint64_t bstep = decltype(b_mn)::value ? 16 * 128 / 16 : 2;
            constexpr uint64_t bblock = decltype(b_mn)::value ? 64 * 128 / 16 : kBlockBytes / 16;
            uint32_t accumulate = 0;
#pragma unroll
            for (int seg = 0; seg < 3; ++seg)
            {
                uint64_t a = smem_desc(smem_u32(seg == 1 ? al : ah), 16, 1024);
                uint64_t b = smem_desc(smem_u32(seg == 0 ? bl : bh), decltype(b_mn)::value ? kBlockBytes : 16, 1024);
#pragma unroll 1
                for (int k = 0; k < terms; k += 64)
                {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                    {
                        if (k + 16 * q < terms)
                        {
                            if (leader) mma(d, a + 2 * q, b + bstep * q, idesc, accumulate);
                            accumulate = 1;
                        }
                    }
                    a += kBlockBytes / 16;
                    b += bblock;
                }
            }
            if (leader) commit(done);
            __syncwarp();
        }
        mbar_wait(done, phase, p.status, abort);
        phase ^= 1;
        fence_after();
    };

    // decoupled decay, then the step along the orthogonalised update
    const auto stepped = [&](float w, float o) { return __fsub_rn(__fsub_rn(w, __fmul_rn(p.decay, w)), __fmul_rn(p.step, o)); };
    for (int k = 0; k < p.steps; ++k)
    {
        // a block's own columns of S = X X^T
        product(ts, xh, xl, xh, xl, std::false_type{}, m16, n16);
        const int c0 = half * 32;
        float v[32];
        uint32_t r[32];
        const auto fetch = [&](uint32_t at, float f) {
            __syncwarp();
            tmem_ld32(at, r);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) * f;
        };
        if constexpr (!CLUSTER)
        {
            if (c0 < m16)
            {
                fetch(ts + lanes + c0, 1.0f / kUnit);
                if (row < m16) put_planes(sh, sl, row, c0, v);
            }
        }
        else
        {
            // The blocks' sums meet: each block leaves its own in the place of S, and after all have, each reads
            // `band` rows of all of them, adds them in rank order and hands their hi and lo to every block.
            const int band = p.band, pitch = m16 + 4;   // lanes write a row each: 16-byte pieces in all banks
            float* const mine = reinterpret_cast<float*>(sh);
            if (c0 < m16)
            {
                fetch(ts + lanes + c0, 1.0f / kUnit);
                if (row < m16)
                {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                    {
                        if (c0 + 4 * q < m16)
                        {
                            *reinterpret_cast<float4*>(mine + row * pitch + c0 + 4 * q) =
                                make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        }
                    }
                }
            }
            pair::cluster_arrive();
            pair::cluster_wait();
            // groups of four columns of this block's rows; at most 4 a thread (64 x 128 / 4 / 512)
            const int rows_here = min(band, m16 - rank * band), s_log = p.s_log, groups = max(0, rows_here) << s_log;
            float sums[4][4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
            {
                const int e = static_cast<int>(threadIdx.x) + q * kSmallThreads;
#pragma unroll
                for (int i = 0; i < 4; ++i) sums[q][i] = 0.0f;
                const int r = e >> s_log, c = (e & ((1 << s_log) - 1)) * 4;
                if (e < groups && c < m16)
                {
                    const float* at = mine + (rank * band + r) * pitch + c;
#pragma unroll 8
                    for (int b = 0; b < ranks; ++b)
                    {
                        float w[4];
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3])
                                     : "r"(pair::peer_addr(at, b)));
#pragma unroll
                        for (int i = 0; i < 4; ++i) sums[q][i] += w[i];
                    }
                }
            }
            pair::cluster_arrive();   // all have read
            pair::cluster_wait();
#pragma unroll
            for (int q = 0; q < 4; ++q)
            {
                const int e = static_cast<int>(threadIdx.x) + q * kSmallThreads;
                const int r = e >> s_log, c = (e & ((1 << s_log) - 1)) * 4;
                if (e < groups && c < m16)
                {
                    uint32_t h[2], l[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                    {
                        h[i] = pack_f16(sums[q][2 * i], sums[q][2 * i + 1]);
                        const float2 back = unpack_f16(h[i]);
                        l[i] = pack_f16(sums[q][2 * i] - back.x, sums[q][2 * i + 1] - back.y);
                    }
                    const uint32_t at = plane_at(rank * band + r, c);
                    for (int b = 0; b < ranks; ++b)
                    {
                        const uint32_t to = pair::peer_addr(sh + at, b);
                        asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(h[0]), "r"(h[1]) : "memory");
                        asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(to + sb * kBlockBytes), "r"(l[0]), "r"(l[1])
                                     : "memory");
                    }
                }
            }
            asm volatile("fence.proxy.async;" ::: "memory");   // the products read S through the other proxy
            pair::cluster_arrive();   // S is everywhere
            pair::cluster_wait();
        }
        product(ts, sh, sl, sh, sl, std::false_type{}, m16, m16);
        if (c0 < m16)
        {
            fetch(ts + lanes + c0, p.cc / kUnit);
            if (row < m16)
            {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                {
                    const uint32_t at = (c0 >> 6) * kBlockBytes + sw128_offset(row, ((c0 & 63) >> 3) + q);
                    const uint4 l4 = *reinterpret_cast<const uint4*>(sl + at), h4 = *reinterpret_cast<const uint4*>(sh + at);
                    const uint32_t l[4] = {l4.x, l4.y, l4.z, l4.w}, h[4] = {h4.x, h4.y, h4.z, h4.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                    {
                        const float2 le = unpack_f16(l[i]), he = unpack_f16(h[i]);
                        v[8 * q + 2 * i] = fmaf(p.cb, he.x, fmaf(p.cb, le.x, v[8 * q + 2 * i]));
                        v[8 * q + 2 * i + 1] = fmaf(p.cb, he.y, fmaf(p.cb, le.y, v[8 * q + 2 * i + 1]));
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = c0 + i == row ? v[i] + p.ca * kUnit : v[i];
                put_planes(sh, sl, row, c0, v);
            }
        }
        product(tx, sh, sl, xh, xl, std::true_type{}, n16, m16);
#pragma unroll 1
        for (int c = c0; c < n16; c += 128)
        {
            fetch(tx + lanes + c, 1.0f / kUnit);
            if (k < p.steps - 1)
            {
                if (row < m16) put_planes(xh, xl, row, c, v);
            }
            else if (row < m)
            {
                // the result waits as fp32 in X's place, rows as the caller's; a wide one's 16-byte groups
                // are turned by their row, since each lane writes to its own
                float* const out = reinterpret_cast<float*>(xh);
                if (tall)
                {
                    float* const to = out + c * m16 + row;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                    {
                        if (c + i < n) to[i * m16] = v[i] * (1.0f / kUnit);
                    }
                }
                else
                {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                    {
                        const int at = row * nb * 64 + (((c + i) / 4) ^ (row & 7)) * 4;
                        *reinterpret_cast<float4*>(out + at) = make_float4(v[i] * (1.0f / kUnit), v[i + 1] * (1.0f / kUnit),
                                                                           v[i + 2] * (1.0f / kUnit), v[i + 3] * (1.0f / kUnit));
                    }
                }
            }
        }
    }
    __syncthreads();
    if (!skip)
    {
        const float* const out = reinterpret_cast<const float*>(xh);
        const int step = p.vec_out ? 4 : 1, out_log = p.out_log, count = own_rows << out_log;
        const int64_t base = p.stride_o * matrix + (tall ? from * p.ldo : from);
        constexpr int kItems = 8;
        for (int e0 = threadIdx.x; e0 < count; e0 += kItems * kSmallThreads)
        {
            float w[MUON ? kItems : 1][4];
            if constexpr (MUON)
            {
#pragma unroll
                for (int q = 0; q < kItems; ++q)
                {
                    const int e = e0 + q * kSmallThreads, r = e >> out_log, c = (e & ((1 << out_log) - 1)) * step;
                    if (e < count && c < own_cols)
                    {
                        const float* at = static_cast<const float*>(p.dst) + base + r * p.ldo + c;
                        if (p.vec_out) load_n<float, 4>(at, w[q]);
                        else w[q][0] = *at;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < kItems; ++q)
            {
                const int e = e0 + q * kSmallThreads, r = e >> out_log, c = (e & ((1 << out_log) - 1)) * step;
                if (q * kSmallThreads >= count - e0) break;
                if (c >= own_cols) continue;
                const int64_t at = base + r * p.ldo + c;
                const float* x = out + (tall ? r * m16 + c : r * nb * 64 + ((c / 4) ^ (r & 7)) * 4 + c % 4);
                float o[4];
                if (p.vec_out)
                {
                    const float4 x4 = *reinterpret_cast<const float4*>(x);
                    o[0] = x4.x, o[1] = x4.y, o[2] = x4.z, o[3] = x4.w;
                }
                else
                {
                    o[0] = *x;
                }
                if constexpr (MUON)
                {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                    {
                        if (k < step) o[k] = stepped(w[q][k], o[k]);
                    }
                    float* to = static_cast<float*>(p.dst) + at;
                    if (p.vec_out) store_four(to, o);
                    else *to = o[0];
                    if (p.lowp != nullptr)
                    {
                        if (p.vec_out) store_four(p.lowp + at, o);
                        else p.lowp[at] = __float2bfloat16_rn(o[0]);
                    }
                }
                else if (p.vec_out)
                {
                    store_four(static_cast<T*>(p.dst) + at, o);
                }
                else
                {
                    static_cast<T*>(p.dst)[at] = from_f32<T>(o[0]);
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    if constexpr (CLUSTER) pair::cluster_sync();   // no block leaves while another may still write to it
    if (warp == 1)
    {
        fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- host ------------------------------------------------------------------------------------
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

constexpr int64_t kMaxExtent = 1 << 20;
constexpr int64_t kMaxBatch = 1 << 15;
constexpr int kMaxSteps = 64;   // the workspace holds counters for as many

struct Layout
{
    int planes;              // of S and P: 1, or 2 for split products
    int64_t m, ldx, plane_x, lds, plane_s;
    unsigned blocks;         // per matrix, of the elementwise launches
    size_t partials, counters, x[2], s, p, total;
};

Layout layout(int64_t batch, int64_t rows, int64_t cols, bool split, int steps)
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
    l.counters = take(batch * 3 * steps * 4);
    l.x[0] = take(batch * 2 * l.plane_x * 2);
    l.x[1] = take(batch * 2 * l.plane_x * 2);
    l.s = take(batch * l.planes * l.plane_s * 2);
    l.p = take(batch * l.planes * l.plane_s * 2);
    l.total = at;
    return l;
}

bool is_small(int64_t rows, int64_t cols)
{
    return std::min(rows, cols) <= kSmallSide && std::max(rows, cols) <= kMaxRanks * kSmallLong;
}

// A block of the small form takes all of an SM's registers (512 threads of more than 120), so no other kernel's blocks
// run beside the allocation of its tensor memory, though its launches overlap.
// Launches the small form; `*taken` stays false where the tiled form is faster, or the device cannot hold a
// cluster of that many blocks.
template <typename T, bool MUON>
int launch_small(const char* what, Small p, int64_t batch, bool split, cudaStream_t stream, bool* taken)
{
    const int smem = small_smem(p);
    const bool cluster = p.ranks > 1;
    const auto kernel = cluster ? small_kernel<T, MUON, true> : small_kernel<T, MUON, false>;
    // per device and cluster size: 0 not asked yet, else 1 + the clusters that run at a time
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices][kMaxRanks + 1];
    int device = 0;
    cudaGetDevice(&device);
    if (device < 0 || device >= kDevices)
    {
        return fail(VEDA_ERR_UNSUPPORTED, std::string(what) + ": no such device");
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(batch * p.ranks));
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = static_cast<unsigned>(p.ranks);
    attrs[0].val.clusterDim.y = 1;
    attrs[0].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 1;
    int room = known[device][p.ranks].load(std::memory_order_acquire);
    if (room == 0)
    {
        constexpr int kMost = 224 * 1024;   // dynamic; a block also has some static shared memory
        bool ok = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) == cudaSuccess;
        if (ok && p.ranks > 8)
        {
            ok = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
        }
        int clusters = 1;
        if (ok && cluster)
        {
            cfg.dynamicSmemBytes = kMost;
            ok = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess;
            cfg.dynamicSmemBytes = smem;
        }
        cudaGetLastError();
        room = ok ? 1 + clusters : 1;
        if (ok)   // an error is not an answer: asked again at the next call
        {
            known[device][p.ranks].store(room, std::memory_order_release);
        }
    }
    // One block a matrix, or smaller sides of at most 64, are always worth it. Of larger ones the
    // tiled form, which fills the device, does more matrices in the time (the more so in bf16, where
    // its products are not split): bf16 64 x 128 x 1024 158 us here and 182 us tiled, 200 of them 570
    // and 505; 8 x 128 x 4096 181 and 205, 64 of them 947 and 618; fp32 32 x 128 x 4096 460 and 565,
    // 64 x 4096 x 128 946 and 694. In all of these the longer side is cut in more than two.
    const int few = split ? 4 : 2;
    *taken = room > 1 && (std::min(p.rows, p.cols) <= 64 || p.ranks <= few || batch <= static_cast<int64_t>(few) * (room - 1));
    if (!*taken)
    {
        return VEDA_OK;
    }
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = overlapped_launches() ? 2 : 1;
    count_launch();
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
    if (err != cudaSuccess)
    {
        cudaGetLastError();
        return fail(VEDA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(err));
    }
    return check_launch(what);
}

// Whether four elements at a time can be read of every row of every matrix.
template <typename T>
bool reads_four(const Source& src, int64_t batch, int64_t cols)
{
    const uintptr_t bases = reinterpret_cast<uintptr_t>(src.g) | reinterpret_cast<uintptr_t>(src.momentum);
    return (bases & (src.momentum != nullptr ? 15u : 4 * sizeof(T) - 1)) == 0 && cols % 4 == 0 && src.ld % 4 == 0 &&
           (batch == 1 || src.stride % 4 == 0);
}

// Whether four elements at a time can be written of every row of the result.
template <typename T>
bool writes_four(const Params& p, int64_t batch, int64_t cols, bool muon)
{
    const uintptr_t size = muon ? 4 : sizeof(T);
    return (reinterpret_cast<uintptr_t>(p.dst) & (4 * size - 1)) == 0 && (reinterpret_cast<uintptr_t>(p.lowp) & 7) == 0 &&
           cols % 4 == 0 && p.ldo % 4 == 0 && (batch == 1 || p.stride_o % 4 == 0);
}

// Tiles of one matrix: of S or M (on and right of the diagonal), and of X.
struct Tiling
{
    int64_t half, whole;
};

Tiling tiling(int64_t rows, int64_t cols, int tn)
{
    const int64_t m = std::min(rows, cols), cols_of_s = (m + tn - 1) / tn;
    Tiling t{0, (rows + 255) / 256 * ((cols + tn - 1) / tn)};
    for (int64_t mb = 0; mb < (m + 255) / 256; ++mb) t.half += cols_of_s - mb * (256 / tn);
    return t;
}

// The products of every step, on 256 x TN tiles; p's destination says what the last one (LAST) writes.
template <bool SPLIT, int LAST, int TN>
int products(const char* what, int64_t batch, int64_t rows, int64_t cols, int steps, float a, float b, float c,
             const Layout& l, char* ws, Params p, cudaStream_t stream)
{
    uint16_t* x[2] = {reinterpret_cast<uint16_t*>(ws + l.x[0]), reinterpret_cast<uint16_t*>(ws + l.x[1])};
    uint16_t* sm[2] = {reinterpret_cast<uint16_t*>(ws + l.s), reinterpret_cast<uint16_t*>(ws + l.p)};
    const bool tall = rows > cols;
    const int64_t m = l.m, sp = l.planes * batch;
    bool ok = pair::make_map3(&p.s, sm[0], 2, false, m, m, sp, l.lds, l.plane_s, 64, TN == pair::kTile ? 128 : 64) &&
              pair::make_map3(&p.m, sm[1], 2, false, m, m, sp, l.lds, l.plane_s, 64, TN == pair::kTile ? 128 : 64) &&
              pair::make_map3(&p.s_out, sm[0], 2, false, m, m, sp, l.lds, l.plane_s, 32, 32, pair::Swizzle::k64) &&
              pair::make_map3(&p.m_out, sm[1], 2, false, m, m, sp, l.lds, l.plane_s, 32, 32, pair::Swizzle::k64) &&
              pair::make_map3(&p.s_out_t, sm[0], 2, false, m, m, sp, l.lds, l.plane_s, 32, 32, pair::Swizzle::kNone) &&
              pair::make_map3(&p.m_out_t, sm[1], 2, false, m, m, sp, l.lds, l.plane_s, 32, 32, pair::Swizzle::kNone);
    for (int k = 0; k < 2; ++k)
    {
        ok = ok &&
             pair::make_map3(&p.xg[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 64,
                             tall || TN < pair::kTile ? 64 : 128) &&
             pair::make_map3(&p.xa[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 64,
                             tall && TN == pair::kTile ? 128 : 64) &&
             pair::make_map3(&p.x_out[k], x[k], 2, false, cols, rows, 2 * batch, l.ldx, l.plane_x, 32, 32,
                             pair::Swizzle::k64);
        p.x[k] = x[k];
    }
    if (!ok)
    {
        return fail(VEDA_ERR_CUDA, std::string(what) + ": tensor map creation failed");
    }
    const Tiling tl = tiling(rows, cols, TN);
    const int64_t half = tl.half, whole = tl.whole, iteration = (2 * half + whole) * batch;
    if (iteration >= (1ll << 30) / steps)
    {
        return fail(VEDA_ERR_INVALID_ARGUMENT, std::string(what) + ": too many tiles");
    }
    p.tall = tall;
    p.rows = static_cast<int>(rows);
    p.cols = static_cast<int>(cols);
    p.side = static_cast<int>(m);
    p.planes = l.planes;
    p.batch = static_cast<int>(batch);
    p.steps = steps;
    p.tn = static_cast<int>((m + TN - 1) / TN);
    p.half = static_cast<int>(half);
    p.whole = static_cast<int>(whole);
    p.sym_tiles = static_cast<int>(half * batch);
    p.iteration = static_cast<int>(iteration);
    p.by_iteration = pair::Divisor(static_cast<uint32_t>(iteration));
    p.by_sym = pair::Divisor(static_cast<uint32_t>(half * batch));
    p.by_half = pair::Divisor(static_cast<uint32_t>(half));
    p.by_whole = pair::Divisor(static_cast<uint32_t>(whole));
    p.by_n = pair::Divisor(static_cast<uint32_t>((cols + TN - 1) / TN));
    p.ca = a;
    p.cb = b;
    p.cc = c;
    p.s_ptr = sm[0];
    p.ldx = l.ldx;
    p.plane_x = l.plane_x;
    p.lds = l.lds;
    p.plane_s = l.plane_s;
    p.counters = reinterpret_cast<unsigned*>(ws + l.counters);
    p.status = device_status_ptr();
    using W = Work<LAST, SPLIT, TN>;
    const int clusters = pair::clusters_available<W, 8, SPLIT>();
    if (clusters < 1)
    {
        return pair::none_available(what, clusters);
    }
    // more clusters than a step of the batch has tiles would only wait
    const int64_t most = std::max(half, whole) * batch;
    return pair::launch_together<W, 8, SPLIT>(what, p, static_cast<int>(std::min<int64_t>(most, clusters)), stream);
}

// Whether Muon's products are split: for fp32 weights, and for matrices of some 30 to 50 rows or columns
// whose other side is too long for a cluster, on which fp16 products come out least exact (fp32 weights off by
// 1.1e-5 at 32 x 4200, 3e-6 at 64; split 4e-8). Larger matrices beside bf16 weights are split where the caller asks
// (VEDA_MUON_FP32_PRODUCTS): their master weights come out 3e-6 off without, and 28 x 2048 x 1024 takes 1.4 against 4.7 ms.
bool muon_split(int64_t rows, int64_t cols, bool lowp) { return !lowp || std::min(rows, cols) <= 64; }

// norm, X, then the products of every step; p's destination says what the last one (LAST) writes.
template <typename T, bool SPLIT, int LAST>
int iterate(const char* what, const Source& src, int64_t batch, int64_t rows, int64_t cols, int steps, float a,
            float b, float c, float eps, char* ws, Params p, cudaStream_t stream)
{
    if (is_small(rows, cols))
    {
        const Small q{src,     static_cast<int>(rows), static_cast<int>(cols), steps,        a,          b,
                      c,       eps,                    p.dst,                  p.ldo,        p.stride_o, p.lowp,
                      p.decay, p.step,                 reads_four<T>(src, batch, cols), writes_four<T>(p, batch, cols, LAST == kMuon),
                      device_status_ptr()};
        bool taken = false;
        const int rc = launch_small<T, LAST == kMuon>(what, q, batch, SPLIT, stream, &taken);
        if (rc != VEDA_OK || taken) return rc;
    }
    const Layout l = layout(batch, rows, cols, SPLIT, kMaxSteps);
    double* partials = reinterpret_cast<double*>(ws + l.partials);
    uint16_t* x0 = reinterpret_cast<uint16_t*>(ws + l.x[0]);
    // the destination by TMA where its base, pitch and stride are multiples of 16 bytes
    const auto fits = [&](const void* base, int es) {
        return aligned16(base) && p.ldo * es % 16 == 0 && (batch == 1 || p.stride_o * es % 16 == 0);
    };
    const int64_t stride = batch == 1 ? rows * p.ldo : p.stride_o;
    const bool f32 = LAST == kMuon || SPLIT;
    p.out_f32 = f32;
    // the split form's chunks leave no room to stage the bf16 weights in
    p.vec = !(SPLIT && p.lowp != nullptr) && fits(p.dst, f32 ? 4 : 2) && (p.lowp == nullptr || fits(p.lowp, 2)) &&
            pair::make_map3(&p.dst_out, p.dst, f32 ? 4 : 2, !f32, cols, rows, batch, p.ldo, stride, 32, 32,
                            f32 ? pair::Swizzle::k128 : pair::Swizzle::k64) &&
            (p.lowp == nullptr || pair::make_map3(&p.lowp_out, p.lowp, 2, true, cols, rows, batch, p.ldo, stride, 32, 32,
                                                  pair::Swizzle::k64));
    const dim3 grid(l.blocks, static_cast<unsigned>(batch));
    const bool four = reads_four<T>(src, batch, cols);
    int rc = launch(what, four ? norm_kernel<T, 4> : norm_kernel<T, 1>, grid, dim3(256), 0, stream, src,
                    static_cast<int>(rows), static_cast<int>(cols), partials);
    if (rc != VEDA_OK) return rc;
    rc = launch(what, four ? init_kernel<T, 4> : init_kernel<T, 1>, grid, dim3(256), 0, stream, src,
                static_cast<int>(rows), static_cast<int>(cols), static_cast<const double*>(partials), eps, x0, l.ldx,
                l.plane_x, reinterpret_cast<unsigned*>(ws + l.counters), steps);
    if (rc != VEDA_OK) return rc;
    // Narrow tiles (256 x 128) have half the latency and one and a half times the operand traffic a flop:
    // they win while the wide ones of X leave the 74 CTA pairs at most about one and a half each (1024 x
    // 1024: 136 against 176 us; 8 x 500 x 1500, 96 wide tiles: 362 against 457; 2048 x 4096, 128: 420
    // against 414; 28 x 1024 x 1024, 448: 992 against 843, both under the power cap). Split products take them always: with wide
    // tiles their folds are not overlapped.
    if constexpr (!SPLIT)
    {
        if (tiling(rows, cols, 256).whole * batch > 110)
        {
            return products<SPLIT, LAST, 256>(what, batch, rows, cols, steps, a, b, c, l, ws, p, stream);
        }
    }
    return products<SPLIT, LAST, 128>(what, batch, rows, cols, steps, a, b, c, l, ws, p, stream);
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
    return ns::layout(batch, rows, cols, dtype == VEDA_F32, ns::kMaxSteps).total;
}

extern "C" size_t veda_muon_step_workspace(int64_t batch, int64_t rows, int64_t cols, int dtype)
{
    return veda_orthogonalize_workspace(batch, rows, cols,
                                        dtype == VEDA_BF16 && ns::muon_split(rows, cols, true) ? VEDA_F32 : dtype);
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
    VEDA_REQUIRE(steps >= 1 && steps <= ns::kMaxSteps, "steps must lie in 1 .. 64");
    VEDA_REQUIRE(eps >= 0.0f, "eps must not be negative");
    if (batch == 0 || rows == 0 || cols == 0)
    {
        return VEDA_OK;
    }
    VEDA_REQUIRE(g != nullptr && out != nullptr, "null pointer");
    const bool split = dtype == VEDA_F32;
    int rc = ns::check_workspace("veda_orthogonalize", workspace, workspace_bytes,
                                 ns::layout(batch, rows, cols, split, ns::kMaxSteps).total);
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
    VEDA_REQUIRE(steps >= 1 && steps <= ns::kMaxSteps, "steps must lie in 1 .. 64");
    if (batch == 0 || rows == 0 || cols == 0)
    {
        return VEDA_OK;
    }
    VEDA_REQUIRE(master != nullptr && momentum != nullptr && grad != nullptr, "null pointer");
    const bool split = ns::muon_split(rows, cols, lowp != nullptr) || (flags & VEDA_MUON_FP32_PRODUCTS) != 0;
    int rc = ns::check_workspace("veda_muon_step", workspace, workspace_bytes,
                                 ns::layout(batch, rows, cols, split, ns::kMaxSteps).total);
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
