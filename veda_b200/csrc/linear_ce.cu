// The loss head in one operator: z = x W^T over the vocabulary, softmax cross-entropy against the
// targets, and the gradients of x and W, without the [rows, vocab] logits ever being stored.
//
// The composition autograd::matmul_nt + autograd::cross_entropy of the reference
// (src/libs/autograd/Variable.cpp:325-346, Loss.cpp:18-103), which keeps logits, log-probabilities
// and probabilities of the whole block. With lse_n = log sum_v exp z_nv and the rows whose target
// is counted:
//   forward   loss_n = lse_n - z_n[t_n], loss = mean over the counted rows. One pass over 256 x 256
//             logit tiles in tensor memory; a thread owns a row and keeps the running maximum and
//             the running sum of exponentials (fp32, log2 units) over a strip of tiles, so a row
//             leaves (max, sum) pairs only, which a second launch merges. Bound by the products, the
//             epilogue under the next tile's: bf16 8192 x 151936 x 1024 1.50 ms (1700 TFLOP/s) called by
//             itself at full clocks, 1.75 ms (1457) in runs, which the power cap holds at some 1400 MHz.
//   backward  q = exp(z - lse) - onehot(t), formed piece by piece of the vocabulary from z computed
//             again (the price of not keeping it), dx = coef q W, dW = coef q^T x with
//             coef = upstream / counted rows. A piece of q stays in L2: the launch that multiplies
//             piece c into dx and dW computes piece c + 1 beside it. Bound by the products too (three
//             of them, one more than with stored logits): the same size 5.8 to 6.2 ms called by itself,
//             6.1 to 6.4 in runs (1260 to 1200 TFLOP/s); forward and backward 7.8 to 8.1 ms.
// q is stored without coef, so its largest entry, about -1 at the target, keeps its bits when
// rounded to bf16 whatever the row count; coef is applied to the fp32 sums. The sums over the
// vocabulary (dx) are held in an fp32 buffer, added piece by piece in order: no atomics meet on an
// element within a launch, so results repeat bit for bit. Where dx has few tiles its sums are cut among
// clusters, one fp32 plane a cut, added in order at the end.
//
// fp32 operands: each is split into two fp16 planes, value 2^e = hi + lo (22 bits, e chosen from the
// largest finite value: of w; of the counted rows of x in the backward; of each row of x in the forward, whose
// lse is every row's, so that a row far larger than the counted ones neither overflows nor costs them
// bits), and a product becomes hi lo + lo hi + hi hi on 256 x 128 tiles
// with three times the k-blocks (pair_mma.cuh); lo lo is below the 22nd bit. fp32 CUDA-core products run at a
// twentieth of the tensor cores' rate, so three tensor products are still far cheaper: 1000 x 10007 x 320
// takes 161 us, forward and backward.
//
// A few rows, which only stream the head, and small problems, which only wait for launches, are computed in fp32
// on the CUDA cores (below), for either dtype.
#include "pair_mma.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cstring>

namespace veda::cuda
{
int* device_status_ptr();

namespace lce
{

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kQScale = 8192.0f;   // of the split q planes: |q| <= 1 becomes at most 2^13

// 2^x with the hardware approximation (relative error ~2^-22; -inf -> 0)
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A logit as a reference in log2 units, rounded up: z log2 e - reference, in one fused operation, is at most 0 then.
// Rounded to nearest, it could be positive by 2^-24 of its size, and 2 to that power infinite above 2^31.
__device__ __forceinline__ float log2_units(float z) { return __fmul_ru(z, kLog2e); }

// Device scalars of a call: what turns a tile's sum into a logit, and the gradients' factors. The
// powers of two stay apart from coef: their product with it could be subnormal where dx is not.
struct Scalars
{
    float z;                // 2^-(ex + ew) of split operands (forward: 2^-ew, ex being each row's own), else 1
    float coef;             // upstream / counted rows
    float unit_dx, unit_dw; // 2^-(13 + ew), 2^-(13 + ex) of split operands, else 1
    float x, w;             // 2^ex, 2^ew of split operands
};

// Which tiles each cluster of a backward launch computes: its tiles of kind k are first[k][cid] up to
// first[k][cid + 1].
constexpr int kMaxClusters = 80;
struct Shares
{
    int first[3][kMaxClusters + 1];
};

struct Params
{
    CUtensorMap x, w;        // operands [rows, dim], [vocab, dim] K-major; plane 1: the lo halves
    CUtensorMap x_mn, w_mn;  // the same, MN-major
    CUtensorMap q_in, q_mn;  // piece of q read by the gradient products
    CUtensorMap q_out;       // piece of q written (store boxes)
    CUtensorMap dx, dw;      // fp32 sums of dx, a plane per split; dW (store boxes)
    int rows, vocab, dim;
    int split;               // operands are pairs of fp16 planes
    int is_bf16;
    int num_m;               // row tiles
    // logits of this launch: vocabulary rows v0 .. v0 + 256 num_n
    int v0, num_n, strip_log2;
    pair::Divisor by_m, by_d;   // num_m, num_d
    // gradient products of this launch: q_in holds vocabulary rows g0 .. g0 + gcols
    int g0, gcols, num_d;
    int dx_tiles, dx_kbs;    // tiles of dx, k-blocks of a split
    pair::Divisor by_dx;     // dx_tiles
    Shares shares;
    int dx_add;              // dx sums: 0 store, 1 add
    int dw_mode;             // 0: from registers; 1: TMA store; 2: TMA add (fp32)
    int dw_f32, dw_beta;
    void* dw_ptr;
    int64_t lddw;
    const Scalars* scalars;
    const int64_t* targets;
    int64_t ignore;
    const float* lse;
    const float* row_scale;  // forward, split: 2^ex of each row of x
    float2* parts;           // [strip slots][rows] running (max, sum)
    float* target_logit;     // [rows]
    unsigned* done;          // cleared for the merge's blocks to count themselves
    int* status;
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b)
{
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ float f16_lo(uint32_t w)
{
    return __low2float(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float f16_hi(uint32_t w)
{
    return __high2float(*reinterpret_cast<const __half2*>(&w));
}

// A row's counted target, -1 for a row that is ignored, out of the vocabulary or past the end.
__device__ __forceinline__ int counted_target(const Params& p, int row)
{
    if (row >= p.rows)
    {
        return -1;
    }
    const int64_t t = p.targets[row];
    return t == p.ignore || t < 0 || t >= p.vocab ? -1 : static_cast<int>(t);
}

// ---- forward: running (max, sum) per row over strips of logit tiles ---------------------------
template <int TN_>
struct StatsWork
{
    using Params = lce::Params;
    static constexpr int TN = TN_, CHAIN = 4;
    struct Tile
    {
        bool skip, first, last, a_mn, b_mn;
        int kbs, mb, nb, slot;
        uint32_t idesc;
    };
    struct State
    {
        float m, s, zs;
        int target;
    };

    // Strips run with the row tile fastest: the clusters working at one time share a few strips of
    // the head, which therefore comes from HBM once, while the rows stay in L2.
    static __device__ __forceinline__ bool tile(const Params& p, int cid, int clusters, int i, Tile& t)
    {
        const int strip = 1 << p.strip_log2, sub = i & (strip - 1);
        t.slot = p.by_m.div(cid + (i >> p.strip_log2) * clusters, t.mb);
        t.nb = (t.slot << p.strip_log2) + sub;
        if (t.nb - sub >= p.num_n)
        {
            return false;
        }
        t.skip = t.nb >= p.num_n;
        t.first = sub == 0;
        t.last = sub == strip - 1 || t.nb == p.num_n - 1;
        t.kbs = (p.dim + pair::kBK - 1) / pair::kBK;
        t.a_mn = t.b_mn = false;
        t.idesc = pair::idesc<TN>(p.is_bf16 != 0, false, false);
        return true;
    }

    static __device__ __forceinline__ void operands(const Params& p, const Tile& t, int rank, pair::Piece& a,
                                                    pair::Piece& b)
    {
        a = {&p.x, 0, t.mb * pair::kTile + rank * 128, 0};
        b = {&p.w, 0, p.v0 + t.nb * TN + rank * (TN / 2), 0};
    }
    static __device__ __forceinline__ void ready(const Params&, const Tile&, volatile int*) {}
    static __device__ __forceinline__ void after(const Params&, const Tile&, int) {}
    static __device__ __forceinline__ void prefetch(const Params& p)
    {
        tc::tma_prefetch(&p.x);
        tc::tma_prefetch(&p.w);
    }

    static __device__ __forceinline__ void before(const Params& p, const Tile& t, State& s, int row0, int,
                                                  pair::Staging&, int lane, volatile int*)
    {
        if (t.first)
        {
            if (t.slot == 0 && t.mb == 0 && row0 + lane == 0)
            {
                *p.done = 0;
            }
            s.m = -INFINITY;
            s.s = 0.0f;
            const int row = t.mb * pair::kTile + row0 + lane;
            s.target = counted_target(p, row);
            s.zs = p.split && row < p.rows ? p.scalars->z / p.row_scale[row] : 1.0f;
        }
    }

    template <int COLS>
    static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, State& s, uint32_t taddr,
                                                    int row0, int col0, pair::Staging&, int lane)
    {
        if (t.mb * pair::kTile + row0 >= p.rows)
        {
            return;
        }
        const int row = t.mb * pair::kTile + row0 + lane;
        const int first = p.v0 + t.nb * TN + col0;
#pragma unroll 1
        for (int c = 0; c < COLS; c += 32)
        {
            const int left = p.vocab - first - c;   // columns of this chunk inside the vocabulary
            if (left <= 0)
            {
                break;
            }
            uint32_t r[32];
            tc::tmem_ld32(taddr + static_cast<uint32_t>(c), r);
            float z[32];
#pragma unroll
            for (int j = 0; j < 32; ++j)
            {
                z[j] = __uint_as_float(r[j]);
            }
            if (p.split)
            {
#pragma unroll
                for (int j = 0; j < 32; ++j) z[j] *= s.zs;
            }
            if (left < 32)
            {
#pragma unroll
                for (int j = 0; j < 32; ++j) z[j] = j < left ? z[j] : -INFINITY;
            }
            const int at = s.target - first - c;
            if (__any_sync(0xFFFFFFFFu, at >= 0 && at < 32))
            {
                float zt = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j) zt = j == at ? z[j] : zt;
                if (at >= 0 && at < 32)
                {
                    p.target_logit[row] = zt;
                }
            }
            float mx[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
            for (int j = 4; j < 32; ++j) mx[j & 3] = fmaxf(mx[j & 3], z[j]);
            const float m = fmaxf(s.m, log2_units(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))));
            // a row of -inf so far: any finite reference gives exponentials of 0, and NaN stays NaN
            const float ref = m == -INFINITY ? 0.0f : m;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[j & 3] += ex2(fmaf(z[j], kLog2e, -ref));
            s.s = s.s * ex2(s.m - ref) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
            s.m = m;
        }
        if (t.last && row < p.rows)
        {
            const int halves = TN / COLS;
            p.parts[static_cast<int64_t>(t.slot * halves + col0 / COLS) * p.rows + row] = make_float2(s.m, s.s);
        }
    }
};

// ---- backward: the next piece of q beside the current piece's two products --------------------
enum GradKind { kDw, kDx, kQ };

template <int TN_>
struct GradWork
{
    using Params = lce::Params;
    static constexpr int TN = TN_, CHAIN = 4;
    struct Tile
    {
        bool skip, a_mn, b_mn;
        int kind, kbs, mb, nb, split;
        uint32_t idesc;
    };
    struct State
    {
        float lse2, keep;
        int target;
    };

    // dW tiles first (k runs over the rows), then dx (over the piece), then q (over dim): Shares gives
    // every cluster the same number of k-blocks as nearly as whole tiles allow.
    static __device__ __forceinline__ bool tile(const Params& p, int cid, int clusters, int i, Tile& t)
    {
        (void)clusters;
        const bool bf = p.is_bf16 != 0;
        t.skip = false;
        int u = p.shares.first[kDw][cid] + i;
        int end = p.shares.first[kDw][cid + 1];
        if (u < end)
        {
            t.kind = kDw;
            t.mb = p.by_d.div(u, t.nb);
            t.kbs = (p.rows + pair::kBK - 1) / pair::kBK;
            t.a_mn = t.b_mn = true;
            t.idesc = pair::idesc<TN>(bf, true, true);
            return true;
        }
        u = p.shares.first[kDx][cid] + (u - end);
        end = p.shares.first[kDx][cid + 1];
        if (u < end)
        {
            t.kind = kDx;
            t.split = p.by_dx.div(u, u);
            t.mb = p.by_d.div(u, t.nb);
            t.kbs = min(p.dx_kbs, (p.gcols + pair::kBK - 1) / pair::kBK - t.split * p.dx_kbs);
            t.a_mn = false;
            t.b_mn = true;
            t.idesc = pair::idesc<TN>(bf, false, true);
            return true;
        }
        u = p.shares.first[kQ][cid] + (u - end);
        end = p.shares.first[kQ][cid + 1];
        if (u >= end)
        {
            return false;
        }
        t.kind = kQ;
        t.nb = p.by_m.div(u, t.mb);
        t.kbs = (p.dim + pair::kBK - 1) / pair::kBK;
        t.a_mn = t.b_mn = false;
        t.idesc = pair::idesc<TN>(bf, false, false);
        return true;
    }

    static __device__ __forceinline__ void operands(const Params& p, const Tile& t, int rank, pair::Piece& a,
                                                    pair::Piece& b)
    {
        const int m = t.mb * pair::kTile + rank * 128, n = t.nb * TN + rank * (TN / 2);
        if (t.kind == kDw)
        {
            a = {&p.q_mn, m, 0, 0};
            b = {&p.x_mn, n, 0, 0};
        }
        else if (t.kind == kDx)
        {
            const int k = t.split * p.dx_kbs * pair::kBK;
            a = {&p.q_in, k, m, 0};
            b = {&p.w_mn, n, p.g0 + k, 0};
        }
        else
        {
            a = {&p.x, 0, m, 0};
            b = {&p.w, 0, p.v0 + n, 0};
        }
    }
    static __device__ __forceinline__ void ready(const Params&, const Tile&, volatile int*) {}
    static __device__ __forceinline__ void after(const Params&, const Tile&, int) {}
    static __device__ __forceinline__ void prefetch(const Params& p)
    {
        tc::tma_prefetch(&p.x);
        tc::tma_prefetch(&p.w);
        tc::tma_prefetch(&p.x_mn);
        tc::tma_prefetch(&p.w_mn);
        tc::tma_prefetch(&p.q_in);
        tc::tma_prefetch(&p.q_mn);
    }

    static __device__ __forceinline__ void before(const Params& p, const Tile& t, State& s, int row0, int,
                                                  pair::Staging&, int lane, volatile int*)
    {
        if (t.kind == kQ)
        {
            const int row = t.mb * pair::kTile + row0 + lane;
            s.target = counted_target(p, row);
            s.lse2 = s.target >= 0 ? p.lse[row] * kLog2e : 0.0f;
        }
    }

    template <int COLS>
    static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, State& s, uint32_t taddr,
                                                    int row0, int col0, pair::Staging& st, int lane)
    {
        if (t.kind == kQ)
        {
            epilogue_q<COLS>(p, t, s, taddr, row0, col0, st, lane);
        }
        else
        {
            epilogue_grad<COLS>(p, t, taddr, row0, col0, st, lane);
        }
    }

    // q of the tile's rows, 64 columns at a time: 0 in ignored rows and past the vocabulary.
    template <int COLS>
    static __device__ __forceinline__ void epilogue_q(const Params& p, const Tile& t, const State& s,
                                                      uint32_t taddr, int row0, int col0, pair::Staging& st,
                                                      int lane)
    {
        const int trow = t.mb * pair::kTile + row0;
        if (trow >= p.rows)
        {
            return;
        }
        const float zs = p.split ? p.scalars->z * kLog2e : kLog2e;
        const float scale = p.split ? kQScale : 1.0f;
#pragma unroll 1
        for (int c = 0; c < COLS; c += 64)
        {
            const int col = t.nb * TN + col0 + c;   // within the piece
            const int left = p.vocab - p.v0 - col;
            uint32_t hi[32], lo[32];
#pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                uint32_t r[32];
                tc::tmem_ld32(taddr + static_cast<uint32_t>(c + 32 * half), r);
                const int at = s.target - p.v0 - col - 32 * half;
                const bool plain = left >= 64 && !__any_sync(0xFFFFFFFFu, s.target < 0 || (at >= 0 && at < 32));
                float q[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) q[j] = ex2(fmaf(__uint_as_float(r[j]), zs, -s.lse2));
                if (!plain)
                {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                    {
                        const float v = j == at ? q[j] - 1.0f : q[j];
                        q[j] = s.target >= 0 && 32 * half + j < left ? v : 0.0f;
                    }
                }
                if (p.split)
                {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                    {
                        const float a = q[2 * j] * scale, b = q[2 * j + 1] * scale;
                        const uint32_t h = pack_f16(a, b);
                        hi[16 * half + j] = h;
                        lo[16 * half + j] = pack_f16(a - f16_lo(h), b - f16_hi(h));
                    }
                }
                else
                {
#pragma unroll
                    for (int j = 0; j < 16; ++j) hi[16 * half + j] = pack_bf16(q[2 * j], q[2 * j + 1]);
                }
            }
            send(p, hi, col, trow, 0, st, lane);
            if (p.split)
            {
                send(p, lo, col, trow, 1, st, lane);
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
            tc::tma_store_3d(&p.q_out, buf, col, row, plane);
            tc::bulk_commit_group();
        }
        st.sent();
    }

    // dx: the fp32 sums as they are. dW: times coef, rounded once to its type.
    template <int COLS>
    static __device__ __forceinline__ void epilogue_grad(const Params& p, const Tile& t, uint32_t taddr,
                                                         int row0, int col0, pair::Staging& st, int lane)
    {
        const bool dw = t.kind == kDw;
        const int trow = t.mb * pair::kTile + row0;   // within the piece for dW
        if (trow >= (dw ? p.gcols : p.rows))
        {
            return;
        }
        const float coef = dw ? p.scalars->coef : 1.0f, unit = dw ? p.scalars->unit_dw : 1.0f;
        const bool f32 = !dw || p.dw_f32;
        const int step = f32 ? 32 : 64;
        const int mode = dw ? p.dw_mode : 1 + p.dx_add;
        const int orow = dw ? p.g0 + trow : trow;
#pragma unroll 1
        for (int c = 0; c < COLS; c += step)
        {
            const int col = t.nb * TN + col0 + c;
            if (col >= p.dim)
            {
                break;
            }
            uint32_t r[32], r2[32];
            tc::tmem_ld32(taddr + static_cast<uint32_t>(c), r);
            if (!f32)
            {
                tc::tmem_ld32(taddr + static_cast<uint32_t>(c + 32), r2);
            }
            if (mode == 0)
            {
                store_direct(p, r, orow, col, p.gcols - trow, unit, coef, st, lane);
                if (!f32)
                {
                    store_direct(p, r2, orow, col + 32, p.gcols - trow, unit, coef, st, lane);
                }
                continue;
            }
            uint8_t* buf = st.buffer(lane);
            if (f32)
            {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    float4 o = make_float4(__uint_as_float(r[4 * k]), __uint_as_float(r[4 * k + 1]),
                                           __uint_as_float(r[4 * k + 2]), __uint_as_float(r[4 * k + 3]));
                    if (dw)
                    {
                        o = make_float4(o.x * unit * coef, o.y * unit * coef, o.z * unit * coef, o.w * unit * coef);
                    }
                    *reinterpret_cast<float4*>(buf + tc::sw128_offset(lane, k)) = o;
                }
            }
            else
            {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    uint32_t w[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                    {
                        const int j = 8 * (k & 3) + 2 * q;
                        const uint32_t a = k < 4 ? r[j] : r2[j], b = k < 4 ? r[j + 1] : r2[j + 1];
                        w[q] = pack_bf16(__uint_as_float(a) * coef, __uint_as_float(b) * coef);
                    }
                    *reinterpret_cast<uint4*>(buf + tc::sw128_offset(lane, k)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0)
            {
                const CUtensorMap* map = dw ? &p.dw : &p.dx;
                const int z = dw ? 0 : t.split;
                if (mode == 2)
                {
                    pair::reduce_add_3d(map, buf, col, orow, z);
                }
                else
                {
                    tc::tma_store_3d(map, buf, col, orow, z);
                }
                tc::bulk_commit_group();
            }
            st.sent();
        }
    }

    // Up to 32 rows of dW whose pitch or base TMA cannot describe, or bf16 accumulation: through the staging, row
    // by row, a column a lane. With a row a lane, each store to 32 lines, 2000 x 30000 x 511 in bf16 took
    // 399 us instead of 305.
    static __device__ __forceinline__ void store_direct(const Params& p, const uint32_t (&r)[32], int row, int col, int rows,
                                                        float unit, float coef, pair::Staging& st, int lane)
    {
        uint8_t* buf = st.buffer(lane);
#pragma unroll
        for (int k = 0; k < 8; ++k)
        {
            *reinterpret_cast<float4*>(buf + tc::sw128_offset(lane, k)) =
                make_float4(__uint_as_float(r[4 * k]) * unit * coef, __uint_as_float(r[4 * k + 1]) * unit * coef,
                            __uint_as_float(r[4 * k + 2]) * unit * coef, __uint_as_float(r[4 * k + 3]) * unit * coef);
        }
        __syncwarp();
        const int n = col + lane < p.dim ? min(32, rows) : 0;
        const int64_t at = static_cast<int64_t>(row) * p.lddw + col + lane;
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 8)
        {
            float old[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                old[i] = 0.0f;
                if (p.dw_beta && i0 + i < n)
                {
                    const int64_t here = at + (i0 + i) * p.lddw;
                    old[i] = p.dw_f32 ? static_cast<const float*>(p.dw_ptr)[here] : __bfloat162float(static_cast<const bf16*>(p.dw_ptr)[here]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                if (i0 + i < n)
                {
                    const int64_t here = at + (i0 + i) * p.lddw;
                    const float v = *reinterpret_cast<const float*>(buf + tc::sw128_offset(i0 + i, lane >> 2) + (lane & 3) * 4);
                    const float o = p.dw_beta ? old[i] + v : v;
                    if (p.dw_f32) static_cast<float*>(p.dw_ptr)[here] = o;
                    else static_cast<bf16*>(p.dw_ptr)[here] = __float2bfloat16_rn(o);
                }
            }
        }
        __syncwarp();
        if (lane == 0) tc::bulk_commit_group();   // empty: the staging counts groups
        st.sent();
    }
};

// ---- the small launches around them ------------------------------------------------------------
constexpr int kMaxBlocks = 296;   // partial maxima of an operand

__device__ __forceinline__ bool counted(int64_t t, int64_t ignore, int64_t vocab)
{
    return t != ignore && t >= 0 && t < vocab;
}

// 2^e that brings a largest magnitude into [2^13, 2^14), clamped so that 2^e and 2^-e are normal
// (a tensor of magnitudes below 2^-113 keeps fewer bits).
__device__ __forceinline__ float split_scale(float top)
{
    if (top == 0.0f)
    {
        return 1.0f;
    }
    int e;
    frexpf(top, &e);   // top = f 2^e, f in [1/2, 1)
    e = 14 - e;
    return ldexpf(1.0f, e < -120 ? -120 : e > 120 ? 120 : e);
}

// Largest finite magnitude of the counted rows of x (blocks below gx) and of w (the others) as one
// partial per block; with row_scale, the scale of every row of x instead of x's partials.
__global__ void __launch_bounds__(256)
absmax_kernel(const float* __restrict__ x, int64_t ldx, int64_t rows, const float* __restrict__ w, int64_t ldw,
              int64_t vocab, int64_t dim, const int64_t* __restrict__ targets, int64_t ignore, int gx,
              float* __restrict__ part, float* __restrict__ row_scale)
{
    __shared__ float warp_part[8];
    dep_wait();
    dep_release();
    const bool is_w = static_cast<int>(blockIdx.x) >= gx;
    const float* m = is_w ? w : x;
    const int64_t ld = is_w ? ldw : ldx, n = is_w ? vocab : rows;
    const int64_t b = is_w ? blockIdx.x - gx : blockIdx.x, blocks = is_w ? gridDim.x - gx : gx;
    const bool by_row = !is_w && row_scale != nullptr;
    float top = 0.0f;
    for (int64_t r = b * 8 + threadIdx.x / 32; r < n; r += blocks * 8)
    {
        if (!is_w && !by_row && !counted(targets[r], ignore, vocab))
        {
            continue;
        }
        for (int64_t c = threadIdx.x & 31; c < dim; c += 32)
        {
            const float v = fabsf(m[r * ld + c]);
            top = v <= FLT_MAX ? fmaxf(top, v) : top;
        }
        if (by_row)
        {
            top = warp_max(top);
            if ((threadIdx.x & 31) == 0) row_scale[r] = split_scale(top);
            top = 0.0f;
        }
    }
    if (by_row)
    {
        return;
    }
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        for (int k = 1; k < 8; ++k) top = fmaxf(top, warp_part[k]);
        part[blockIdx.x] = top;
    }
}

// What comes before the tensor-core launches, in one: the call's scalars (the last block: split scales
// from the partial maxima, upstream / counted rows) and the operand planes of x (blocks below gx) and w
// (the next gw) with a pitch of a multiple of 8 elements: a bf16 copy, or the two fp16 halves of an fp32
// operand. clear: rows of x that are not counted become zeros, so that what padding holds (NaN
// included) meets q = 0 in dW's product as 0. vx, vw: eight elements of a row can be read at a time. row_scale: the
// scales of the rows of x, if each has its own (parts_x is 0 then).
template <typename T>
__global__ void __launch_bounds__(256)
pack_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, const T* __restrict__ w, int64_t ldw, int64_t vocab,
            int64_t dim, const int64_t* __restrict__ targets, int64_t ignore, bool clear, bool vx, bool vw, int gx, int gw,
            uint16_t* __restrict__ px, uint16_t* __restrict__ pw, int64_t ldp, const float* __restrict__ part, int first_w,
            int parts_x, int parts_w, const float* __restrict__ row_scale, const float* __restrict__ upstream, Scalars* __restrict__ scalars, int* status)
{
    __shared__ int counts[8];
    __shared__ float tops[2][8];
    __shared__ float scale_shared[2];
    dep_wait();
    dep_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int block = static_cast<int>(blockIdx.x);
    if (part != nullptr)
    {
        float tx = 0.0f, tw = 0.0f;
        for (int i = threadIdx.x; i < parts_x; i += 256) tx = fmaxf(tx, part[i]);
        for (int i = threadIdx.x; i < parts_w; i += 256) tw = fmaxf(tw, part[first_w + i]);
        tx = warp_max(tx);
        tw = warp_max(tw);
        if (lane == 0) tops[0][warp] = tx, tops[1][warp] = tw;
        __syncthreads();
        if (threadIdx.x < 2)
        {
            float top = 0.0f;
            for (int k = 0; k < 8; ++k) top = fmaxf(top, tops[threadIdx.x][k]);
            scale_shared[threadIdx.x] = split_scale(top);
        }
        __syncthreads();
    }
    if (block == gx + gw)
    {
        int n = 0, bad = 0;
        for (int64_t i = threadIdx.x; i < rows; i += 256)
        {
            const int64_t t = targets[i];
            if (t != ignore)
            {
                t >= 0 && t < vocab ? ++n : ++bad;
            }
        }
        n = __reduce_add_sync(0xFFFFFFFFu, n);
        if (__any_sync(0xFFFFFFFFu, bad != 0) && lane == 0 && status != nullptr)
        {
            *status = VEDA_ERR_OUT_OF_RANGE;
        }
        if (lane == 0) counts[warp] = n;
        __syncthreads();
        if (threadIdx.x == 0)
        {
            int total = 0;
            for (int k = 0; k < 8; ++k) total += counts[k];
            // no counted row: the loss and every gradient are zero
            const float coef = total > 0 ? (upstream != nullptr ? *upstream : 1.0f) / static_cast<float>(total) : 0.0f;
            Scalars s{1.0f, coef, 1.0f, 1.0f, 1.0f, 1.0f};
            if (part != nullptr)
            {
                s.x = scale_shared[0];
                s.w = scale_shared[1];
                s.z = 1.0f / s.x / s.w;
                s.unit_dx = 1.0f / kQScale / s.w;
                s.unit_dw = 1.0f / kQScale / s.x;
            }
            *scalars = s;
        }
        return;
    }
    const bool is_w = block >= gx;
    const T* m = is_w ? w : x;
    uint16_t* out = is_w ? pw : px;
    const int64_t ld = is_w ? ldw : ldx, n = is_w ? vocab : rows;
    const int64_t b = is_w ? block - gx : block, blocks = is_w ? gw : gx;
    const float scale = part != nullptr ? scale_shared[is_w ? 1 : 0] : 1.0f;
    const bool by_row = !is_w && row_scale != nullptr;
    const bool vec = is_w ? vw : vx;
    const int64_t per_row = ldp / 8, groups = n * per_row;   // of eight columns
#pragma unroll 2
    for (int64_t g = b * 256 + threadIdx.x; g < groups; g += blocks * 256)
    {
        const int64_t r = g / per_row, c = (g - r * per_row) * 8;
        const int left = static_cast<int>(dim - c < 8 ? dim - c : 8);
        float v[8];
        if (!is_w && clear && !counted(targets[r], ignore, vocab))
        {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = 0.0f;
        }
        else if (vec && left == 8)
        {
            if constexpr (sizeof(T) == 2)
            {
                load16(m + r * ld + c, v);
            }
            else
            {
                float a[4], d[4];
                load16(m + r * ld + c, a);
                load16(m + r * ld + c + 4, d);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = d[k];
            }
        }
        else
        {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < left ? to_f32(m[r * ld + c + k]) : 0.0f;
        }
        uint32_t hi[4], lo[4];
        const float own = by_row ? row_scale[r] : scale;
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            if constexpr (sizeof(T) == 2)
            {
                hi[k] = pack_bf16(v[2 * k], v[2 * k + 1]);   // bf16 values: exact
            }
            else
            {
                const float a = v[2 * k] * own, d = v[2 * k + 1] * own;
                hi[k] = pack_f16(a, d);
                lo[k] = pack_f16(a - f16_lo(hi[k]), d - f16_hi(hi[k]));
            }
        }
        *reinterpret_cast<uint4*>(out + r * ldp + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (sizeof(T) == 4)
        {
            *reinterpret_cast<uint4*>(out + (n + r) * ldp + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
}

// Merges each row's (max, sum) pairs, lse = ln 2 (max + log2 sum), loss = lse - z[target]; the block
// that finishes last takes the mean over the counted rows, in double and in a fixed order (0 when none
// is counted). A block has `width` rows (a power of two) and 256 / width threads a row.
__global__ void __launch_bounds__(256)
merge_kernel(const float2* __restrict__ parts, int slots, int64_t rows, int64_t vocab, int width,
             const int64_t* __restrict__ targets, int64_t ignore, const float* __restrict__ target_logit,
             float* row_loss, float* __restrict__ lse, float* loss, unsigned* done, int* status)
{
    __shared__ float2 part[256];
    __shared__ double sums[8];
    __shared__ int counts[8];
    __shared__ bool last;
    dep_wait();
    dep_release();
    const int tid = static_cast<int>(threadIdx.x), mine = tid & (width - 1), slice = tid / width, slices = 256 / width;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * width + mine;
    float m = -INFINITY, s = 0.0f;
    auto add = [&](float2 o) {
        const float top = fmaxf(m, o.x);
        const float ref = top == -INFINITY ? 0.0f : top;
        s = s * ex2(m - ref) + o.y * ex2(o.x - ref);
        m = top;
    };
    if (row < rows)
    {
#pragma unroll 4
        for (int k = slice; k < slots; k += slices) add(parts[static_cast<int64_t>(k) * rows + row]);
    }
    int top = slices;
    while (top / 2 >= slots) top /= 2;   // the slices beyond the slots have nothing
    for (int d = top / 2; d > 0; d /= 2)
    {
        part[tid] = make_float2(m, s);
        __syncthreads();
        if (slice < d) add(part[tid + d * width]);
        __syncthreads();
    }
    if (slice == 0 && row < rows)
    {
        // a sum of 0: every term vanished against the rounding of a maximum past 2^31, whose logarithm the sum's
        // could not change
        const float l = (s == 0.0f ? m : m + log2f(s)) * kLn2;
        if (lse != nullptr) lse[row] = l;
        const int64_t t = targets[row];
        const bool inside = t >= 0 && t < vocab;
        if (t != ignore && !inside && status != nullptr)
        {
            *status = VEDA_ERR_OUT_OF_RANGE;
        }
        row_loss[row] = t != ignore && inside ? l - target_logit[row] : 0.0f;
    }
    if (loss == nullptr)
    {
        return;
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(done, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last)
    {
        return;
    }
    __threadfence();
    double sum = 0.0;
    int n = 0;
#pragma unroll 4
    for (int64_t i = tid; i < rows; i += 256)
    {
        if (counted(targets[i], ignore, vocab))
        {
            sum += static_cast<double>(__ldcg(row_loss + i));
            ++n;
        }
    }
    sum = warp_sum(sum);
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    if ((tid & 31) == 0) sums[tid >> 5] = sum, counts[tid >> 5] = n;
    __syncthreads();
    if (tid == 0)
    {
        for (int k = 1; k < 8; ++k) sum += sums[k], n += counts[k];
        *loss = n > 0 ? static_cast<float>(sum / n) : 0.0f;
    }
}

// dx = coef x the fp32 sums, those of the splits added in their order: eight columns a thread, where
// rows allow it.
template <typename T>
__global__ void __launch_bounds__(256)
finish_dx_kernel(const float* __restrict__ acc, int64_t lda, int splits, T* __restrict__ dx, int64_t lddx, int64_t rows,
                 int64_t dim, bool vec, const Scalars* __restrict__ scalars)
{
    dep_wait();
    dep_release();
    const float coef = scalars->coef, unit = scalars->unit_dx;
    const int64_t per_row = (dim + 7) / 8, groups = rows * per_row;
    for (int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; g < groups; g += static_cast<int64_t>(gridDim.x) * 256)
    {
        const int64_t r = g / per_row, c = (g - r * per_row) * 8;
        const float* from = acc + r * lda + c;
        T* to = dx + r * lddx + c;
        if (vec && c + 8 <= dim)
        {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k += 4)
            {
                float a[4];
                load16(from + k, a);
                for (int q = 1; q < splits; ++q)
                {
                    float more[4];
                    load16(from + q * rows * lda + k, more);
#pragma unroll
                    for (int i = 0; i < 4; ++i) a[i] += more[i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) v[k + i] = a[i] * unit * coef;
            }
            constexpr int V = 16 / sizeof(T);
#pragma unroll
            for (int k = 0; k < 8; k += V)
            {
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = v[k + i];
                store16(to + k, o);
            }
        }
        else
        {
            for (int k = 0; k < 8 && c + k < dim; ++k)
            {
                float a = from[k];
                for (int q = 1; q < splits; ++q) a += from[q * rows * lda + k];
                to[k] = from_f32<T>(a * unit * coef);
            }
        }
    }
}

// The same for a small dx of many splits: 32 columns of a row per block, a warp an eighth of the splits.
template <typename T>
__global__ void __launch_bounds__(256)
finish_splits_kernel(const float* __restrict__ acc, int64_t lda, int splits, T* __restrict__ dx, int64_t lddx, int64_t rows,
                     int64_t dim, const Scalars* __restrict__ scalars)
{
    __shared__ float part[8][32];
    dep_wait();
    dep_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane, r = blockIdx.y;
    float sum = 0.0f;
    if (c < dim)
    {
#pragma unroll 4
        for (int k = warp; k < splits; k += 8) sum += acc[(k * rows + r) * lda + c];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < dim)
    {
        for (int k = 1; k < 8; ++k) sum += part[k][lane];
        dx[r * lddx + c] = from_f32<T>(sum * scalars->unit_dx * scalars->coef);
    }
}

// ---- up to four rows: the head streamed past the rows on the CUDA cores -------------------------
// A few rows against the whole head are bound by reading it (and writing dW), not by the products: the
// 256-row tensor tiles would read it at half of HBM's rate and compute mostly padding. Here the rows
// stay in shared memory in fp32, a warp takes four vocabulary rows at a time, 16 bytes a lane and row,
// and keeps 4 x R dot products; sums are fp32 for either dtype and nothing is laid out anew. Backward
// reads the head once: a chunk of vocabulary rows waits in shared memory while its q are formed and
// while dx and dW, each thread its own eight columns, are made of them.
constexpr int kFewRows = 4;
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewBlocks = 4 * 148;   // partial results are kept per block
// Blocks an SM holds, by the registers that R rows take.
constexpr int few_fwd_per_sm(int r) { return r == 1 ? 4 : r == 2 ? 3 : 2; }
constexpr int kFewBwdPerSm = 2;

struct Few
{
    const void *x, *w;
    int64_t ldx, ldw;
    int rows, dim, padded;   // padded: dim rounded up to 256
    int64_t vocab;
    const int64_t* targets;
    int64_t ignore;
    int grain;               // elements of a head row that can be read at a time: 8, or up to 16 bytes of 4, 2 or 1
    // forward
    float2* parts;           // [block][rows]
    float* target_logit;
    // backward
    const float* lse;
    const float* upstream;
    int chunk;               // vocabulary rows held at a time
    void* dw;
    int64_t lddw;
    int dw_f32, dw_beta, dw_grain;   // dw_grain: as grain, of dW's rows; 8 does not ask for whole groups of columns
    float* acc;              // [block][rows][ld_acc] sums of dx, or null
    int64_t ld_acc;
    // small problems
    float* q;                // [rows][vocab]
    void* dx;
    int64_t lddx;
    unsigned* done;
    int* status;
};

// Eight elements of a head row, as they lie: 16 bytes of bf16, 32 of fp32. From global memory they are
// read once and not kept in L1.
template <typename T>
struct Eight
{
    uint4 q[sizeof(T) / 2];
    __device__ __forceinline__ void stream(const T* p)
    {
#pragma unroll
        for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k)
        {
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(q[k].x), "=r"(q[k].y), "=r"(q[k].z), "=r"(q[k].w)
                         : "l"(reinterpret_cast<const uint4*>(p) + k));
        }
    }
    __device__ __forceinline__ void read(const T* p)
    {
#pragma unroll
        for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k) q[k] = reinterpret_cast<const uint4*>(p)[k];
    }
    // G elements at a time, the first `left` (a multiple of G)
    template <int G>
    __device__ __forceinline__ void gather(const T* p, int left)
    {
        struct alignas(G * sizeof(T)) Group
        {
            T v[G];
        };
        Group g[8 / G];
#pragma unroll
        for (int k = 0; k < 8 / G; ++k)
        {
            if (k * G < left)
            {
                g[k] = reinterpret_cast<const Group*>(p)[k];
            }
            else
            {
#pragma unroll
                for (int i = 0; i < G; ++i) g[k].v[i] = from_f32<T>(0.0f);
            }
        }
        memcpy(q, g, sizeof(g));
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k) q[k] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const
    {
        if constexpr (sizeof(T) == 2)
        {
            const uint32_t w[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
        else
        {
#pragma unroll
            for (int k = 0; k < 2; ++k)
            {
                v[4 * k] = __uint_as_float(q[k].x);
                v[4 * k + 1] = __uint_as_float(q[k].y);
                v[4 * k + 2] = __uint_as_float(q[k].z);
                v[4 * k + 3] = __uint_as_float(q[k].w);
            }
        }
    }
};

// The rows in fp32, zero past dim, past the rows and (clear) where a row is not counted; two planes of
// four columns out of eight, so that a warp's 16-byte reads meet no bank twice.
template <typename T, int R>
__device__ __forceinline__ void stage_rows(const Few& p, int r0, float* xs, bool clear)
{
    const T* x = static_cast<const T*>(p.x);
    bool keep[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
    {
        const int row = r0 + r;
        keep[r] = row < p.rows && !(clear && !counted(p.targets[row < p.rows ? row : 0], p.ignore, p.vocab));
    }
    for (int c = threadIdx.x; c < p.padded; c += kFewThreads)
    {
        // all rows' loads before the first store to shared memory, which they could not pass
        float v[R];
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = keep[r] && c < p.dim ? to_f32(x[(r0 + r) * p.ldx + c]) : 0.0f;
        float* at = xs + (c & 4 ? p.padded / 2 : 0) + (c >> 3) * 4 + (c & 3);
#pragma unroll
        for (int r = 0; r < R; ++r) at[r * p.padded] = v[r];
    }
}

// acc[j][r] += the dot product of the lane's columns c .. c + 7 of four head rows and of row r.
template <typename T, int R>
__device__ __forceinline__ void dot8(const Eight<T> (&raw)[4], const float* xs, int padded, int c, float (&acc)[4][R])
{
    float w[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j].values(w[j]);
#pragma unroll
    for (int r = 0; r < R; ++r)
    {
        const float4 a = *reinterpret_cast<const float4*>(xs + r * padded + (c >> 3) * 4);
        const float4 b = *reinterpret_cast<const float4*>(xs + r * padded + padded / 2 + (c >> 3) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            float s = acc[j][r];
            s = fmaf(w[j][0], a.x, s), s = fmaf(w[j][1], a.y, s), s = fmaf(w[j][2], a.z, s), s = fmaf(w[j][3], a.w, s);
            s = fmaf(w[j][4], b.x, s), s = fmaf(w[j][5], b.y, s), s = fmaf(w[j][6], b.z, s), s = fmaf(w[j][7], b.w, s);
            acc[j][r] = s;
        }
    }
}

// The lane's row (lane < R) of four summed dot products.
template <int R>
__device__ __forceinline__ void own_row(float (&acc)[4][R], int lane, float (&z)[4])
{
#pragma unroll
    for (int j = 0; j < 4; ++j)
    {
        z[j] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
        {
            const float s = warp_sum(acc[j][r]);
            z[j] = lane == r ? s : z[j];
        }
    }
}

// blockIdx.y: which R rows. G: the head's grain. Q: writes q of the rows instead of their (max, sum) pairs.
template <typename T, int R, int G, bool Q>
__global__ void __launch_bounds__(kFewThreads, few_fwd_per_sm(R))
few_fwd_kernel(const Few p)
{
    extern __shared__ float few_smem[];
    __shared__ float2 part[kFewWarps][R];
    float* xs = few_smem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r0 = static_cast<int>(blockIdx.y) * R, row_ = r0 + lane;
    dep_wait();
    dep_release();
    if (!Q && p.done != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    {
        *p.done = 0;
    }
    stage_rows<T, R>(p, r0, xs, false);
    __syncthreads();
    const bool own = lane < R && row_ < p.rows;
    const int64_t target = own ? p.targets[row_] : -1;
    const bool valid = own && counted(target, p.ignore, p.vocab);
    const float lse2 = Q && valid ? p.lse[row_] * kLog2e : 0.0f;
    float m = -INFINITY, s = 0.0f;
    for (int64_t v = (static_cast<int64_t>(blockIdx.x) * kFewWarps + warp) * 4; v < p.vocab;
         v += static_cast<int64_t>(gridDim.x) * kFewWarps * 4)
    {
        const T* row[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) row[j] = static_cast<const T*>(p.w) + (v + j < p.vocab ? v + j : v) * p.ldw;
        float acc[4][R] = {};
        // two chunks of columns at a time, all their loads first
        for (int c = lane * 8; c < p.padded; c += 512)
        {
            Eight<T> w[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                const int at = c + 256 * h;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    if constexpr (G == 8)
                    {
                        w[h][j].zero();
                        if (at < p.dim) w[h][j].stream(row[j] + at);
                    }
                    else
                    {
                        w[h][j].template gather<G>(row[j] + at, p.dim - at);
                    }
                }
            }
            dot8<T, R>(w[0], xs, p.padded, c, acc);
            if (c + 256 < p.padded) dot8<T, R>(w[1], xs, p.padded, c + 256, acc);
        }
        float z[4];
        own_row<R>(acc, lane, z);
        if constexpr (Q)
        {
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                if (own && v + j < p.vocab)
                {
                    const float q = ex2(fmaf(z[j], kLog2e, -lse2)) - (target == v + j ? 1.0f : 0.0f);
                    p.q[row_ * p.vocab + v + j] = valid ? q : 0.0f;
                }
            }
        }
        else
        {
            float top = m;
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                if (v + j >= p.vocab) z[j] = -INFINITY;
                else if (valid && target == v + j) p.target_logit[row_] = z[j];
                top = fmaxf(top, log2_units(z[j]));
            }
            const float ref = top == -INFINITY ? 0.0f : top;
            s *= ex2(m - ref);
#pragma unroll
            for (int j = 0; j < 4; ++j) s += ex2(fmaf(z[j], kLog2e, -ref));
            m = top;
        }
    }
    if constexpr (!Q)
    {
        if (lane < R) part[warp][lane] = make_float2(m, s);
        __syncthreads();
        if (warp == 0 && own)
        {
            for (int k = 1; k < kFewWarps; ++k)
            {
                const float2 o = part[k][lane];
                const float top = fmaxf(m, o.x);
                const float ref = top == -INFINITY ? 0.0f : top;
                s = s * ex2(m - ref) + o.y * ex2(o.x - ref);
                m = top;
            }
            p.parts[static_cast<int64_t>(blockIdx.x) * p.rows + row_] = make_float2(m, s);
        }
    }
}

// Copies vocabulary rows v .. v + chunk - 1, as far as there are, into `stage` (rows of `padded` elements), a
// row a warp at a time: asynchronously by 16, 8 or 4 bytes. Single bf16 elements, which nothing copies
// asynchronously, go through registers, 16 loads of a lane at a time. Columns past dim stay as they are.
template <typename T, int BYTES>
__device__ __forceinline__ void stage_async(const Few& p, T* stage, int64_t v)
{
    constexpr int G = BYTES / sizeof(T);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < p.chunk && v + r < p.vocab; r += kFewWarps)
    {
        const T* row = static_cast<const T*>(p.w) + (v + r) * p.ldw;
        const uint32_t to = tc::smem_u32(stage + r * p.padded);
        for (int c = lane * G; c < p.dim; c += 32 * G)
        {
            if constexpr (BYTES == 16)
            {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + c * static_cast<int>(sizeof(T))), "l"(row + c) : "memory");
            }
            else
            {
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to + c * static_cast<int>(sizeof(T))), "l"(row + c), "n"(BYTES)
                             : "memory");
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void stage_head(const Few& p, T* stage, int64_t v)
{
    const int bytes = p.grain * static_cast<int>(sizeof(T));
    if (bytes >= 16)
    {
        stage_async<T, 16>(p, stage, v);
    }
    else if (bytes == 8)
    {
        stage_async<T, 8>(p, stage, v);
    }
    else if (bytes == 4)
    {
        stage_async<T, 4>(p, stage, v);
    }
    else
    {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int r0 = warp; r0 < p.chunk; r0 += 4 * kFewWarps)
        {
            for (int c0 = lane; c0 < p.dim; c0 += 128)
            {
                T e[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    const int r = r0 + i * kFewWarps;
                    const T* row = static_cast<const T*>(p.w) + (v + r) * p.ldw;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                    {
                        const bool in = r < p.chunk && v + r < p.vocab && c0 + 32 * k < p.dim;
                        e[i][k] = in ? row[c0 + 32 * k] : from_f32<T>(0.0f);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                    {
                        const int r = r0 + i * kFewWarps;
                        if (r < p.chunk && c0 + 32 * k < p.dim) stage[r * p.padded + c0 + 32 * k] = e[i][k];
                    }
                }
            }
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// Eight columns of a dW row (the first `left` of them), accumulated with beta.
template <int G, typename U>
__device__ __forceinline__ void store_dw_by(U* at, const float (&o)[8], int beta, int left)
{
    struct alignas(G * sizeof(U)) Group
    {
        U v[G];
    };
#pragma unroll
    for (int k = 0; k < 8; k += G)
    {
        if (k < left)
        {
            Group g;
            if (beta) g = *reinterpret_cast<const Group*>(at + k);
#pragma unroll
            for (int i = 0; i < G; ++i) g.v[i] = from_f32<U>(beta ? to_f32(g.v[i]) + o[k + i] : o[k + i]);
            *reinterpret_cast<Group*>(at + k) = g;
        }
    }
}
template <typename U>
__device__ __forceinline__ void store_dw(U* at, const float (&o)[8], int grain, int beta, int left)
{
    constexpr int V = 16 / sizeof(U);
    if (grain == 8 && left >= 8) store_dw_by<V>(at, o, beta, left);
    else if (grain == 4) store_dw_by<4>(at, o, beta, left);
    else if (grain == 2) store_dw_by<2>(at, o, beta, left);
    else store_dw_by<1>(at, o, beta, left);
}

template <typename T, int R>
__global__ void __launch_bounds__(kFewThreads, kFewBwdPerSm)
few_bwd_kernel(const Few p)
{
    extern __shared__ float few_smem[];
    __shared__ float coef_shared;
    float* xs = few_smem;
    float* qs = xs + R * p.padded;                                  // [chunk][R]
    T* stage = reinterpret_cast<T*>(qs + 32 * R);                   // two chunks of head rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    dep_wait();
    dep_release();
    const int64_t step = static_cast<int64_t>(gridDim.x) * p.chunk;
    int64_t v = static_cast<int64_t>(blockIdx.x) * p.chunk;
    for (int r = warp; r < 2 * p.chunk; r += kFewWarps)
    {
        for (int c = p.dim + lane; c < p.padded; c += 32) stage[r * p.padded + c] = from_f32<T>(0.0f);
    }
    if (v < p.vocab) stage_head<T>(p, stage, v);
    stage_rows<T, R>(p, 0, xs, true);
    if (threadIdx.x == 0)
    {
        int n = 0;
        for (int r = 0; r < p.rows; ++r)
        {
            const int64_t t = p.targets[r];
            if (counted(t, p.ignore, p.vocab)) ++n;
            else if (t != p.ignore && p.status != nullptr) *p.status = VEDA_ERR_OUT_OF_RANGE;
        }
        coef_shared = n > 0 ? (p.upstream != nullptr ? *p.upstream : 1.0f) / static_cast<float>(n) : 0.0f;
    }
    const int64_t target = lane < p.rows ? p.targets[lane] : -1;
    const bool valid = lane < p.rows && counted(target, p.ignore, p.vocab);
    const float lse2 = valid ? p.lse[lane] * kLog2e : 0.0f;
    __syncthreads();
    const float coef = coef_shared;
    // eight columns a thread; the threads that are left over take other rows of the chunk
    const int groups = (p.dim + 7) / 8;
    const int share = groups < kFewThreads ? kFewThreads / groups : 1;   // threads per eight columns
    const int mine = threadIdx.x / groups;                               // which of them (>= share: none)
    const int col0 = (threadIdx.x - mine * groups) * 8;
    float dx[R][8] = {};
    for (int buf = 0; v < p.vocab; v += step, buf ^= 1)
    {
        T* const here = stage + buf * p.chunk * p.padded;
        if (v + step < p.vocab) stage_head<T>(p, stage + (buf ^ 1) * p.chunk * p.padded, v + step);
        else asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        // q of four head rows a warp at a time
        for (int r0 = warp * 4; r0 < p.chunk; r0 += kFewWarps * 4)
        {
            float acc[4][R] = {};
            for (int c = lane * 8; c < p.padded; c += 256)
            {
                Eight<T> w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j].read(here + (r0 + j) * p.padded + c);
                dot8<T, R>(w, xs, p.padded, c, acc);
            }
            float z[4];
            own_row<R>(acc, lane, z);
            if (lane < R)
            {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const float q = ex2(fmaf(z[j], kLog2e, -lse2)) - (target == v + r0 + j ? 1.0f : 0.0f);
                    qs[(r0 + j) * R + lane] = valid && v + r0 + j < p.vocab ? q : 0.0f;
                }
            }
        }
        __syncthreads();
        for (int col = col0; mine < share && col < p.dim; col += kFewThreads * 8)
        {
            float x8[R][8];
            if (p.dw != nullptr)
            {
#pragma unroll
                for (int r = 0; r < R; ++r)
                {
                    const float4 a = *reinterpret_cast<const float4*>(xs + r * p.padded + (col >> 3) * 4);
                    const float4 b = *reinterpret_cast<const float4*>(xs + r * p.padded + p.padded / 2 + (col >> 3) * 4);
                    x8[r][0] = a.x, x8[r][1] = a.y, x8[r][2] = a.z, x8[r][3] = a.w;
                    x8[r][4] = b.x, x8[r][5] = b.y, x8[r][6] = b.z, x8[r][7] = b.w;
                }
            }
            for (int k = mine; k < p.chunk && v + k < p.vocab; k += share)
            {
                float q[R];
#pragma unroll
                for (int r = 0; r < R; ++r) q[r] = qs[k * R + r];
                if (p.acc != nullptr)
                {
                    Eight<T> raw;
                    raw.read(here + k * p.padded + col);
                    float w[8];
                    raw.values(w);
#pragma unroll
                    for (int r = 0; r < R; ++r)
                    {
#pragma unroll
                        for (int i = 0; i < 8; ++i) dx[r][i] = fmaf(q[r], w[i], dx[r][i]);
                    }
                }
                if (p.dw != nullptr)
                {
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                    {
                        float sum = 0.0f;
#pragma unroll
                        for (int r = 0; r < R; ++r) sum = fmaf(q[r], x8[r][i], sum);
                        o[i] = sum * coef;
                    }
                    const int64_t at = (v + k) * p.lddw + col;
                    if (p.dw_f32) store_dw(static_cast<float*>(p.dw) + at, o, p.dw_grain, p.dw_beta, p.dim - col);
                    else store_dw(static_cast<bf16*>(p.dw) + at, o, p.dw_grain, p.dw_beta, p.dim - col);
                }
            }
        }
        __syncthreads();   // the chunk and its q are free
    }
    if (p.acc == nullptr)
    {
        return;
    }
    // The sums of the threads that share columns meet in shared memory, in order. A block holds one set
    // of columns per thread, so dim <= 2048 (checked on the host).
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    for (int k = 0; k < share; ++k)
    {
        __syncthreads();
        if (mine == k && col0 < p.dim)
        {
#pragma unroll
            for (int r = 0; r < R; ++r)
            {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                {
                    float* at = xs + r * p.padded + col0 + i;   // x is no longer needed
                    *at = k == 0 ? dx[r][i] : *at + dx[r][i];
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.rows * p.dim; i += kFewThreads)
    {
        const int r = i / p.dim, c = i - r * p.dim;
        p.acc[(static_cast<int64_t>(blockIdx.x) * p.rows + r) * p.ld_acc + c] = xs[r * p.padded + c];
    }
}

// dx = coef x the sum of the blocks' parts: 32 columns of a row per block, eight warps a share each.
template <typename T>
__global__ void __launch_bounds__(256)
few_dx_kernel(const Few p, int blocks, T* __restrict__ dx, int64_t lddx)
{
    __shared__ float part[8][32];
    dep_wait();
    dep_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * 32 + lane, r = blockIdx.y;
    float sum = 0.0f;
    if (c < p.dim)
    {
#pragma unroll 8
        for (int b = warp; b < blocks; b += 8) sum += p.acc[(static_cast<int64_t>(b) * p.rows + r) * p.ld_acc + c];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.dim)
    {
        for (int k = 1; k < 8; ++k) sum += part[k][lane];
        int n = 0;
        for (int k = 0; k < p.rows; ++k) n += counted(p.targets[k], p.ignore, p.vocab) ? 1 : 0;
        const float coef = n > 0 ? (p.upstream != nullptr ? *p.upstream : 1.0f) / static_cast<float>(n) : 0.0f;
        dx[r * lddx + c] = from_f32<T>(sum * coef);
    }
}

// ---- small problems: fp32 products on the CUDA cores --------------------------------------------
// For these (is_small has the rule) the tensor-core path is all launch latency: fp32 128 x 512 x 64 takes nine
// launches and 34 us there. Such a problem takes four here, 23 us: the pairs and their merge as above, rows in
// groups of four, then q, kept in fp32, and both products in 32 x 32 tiles.
constexpr int kSmallTerms = 128;

// Blocks below gx: tiles of dx = coef q W; the others: of dW = coef q^T x. Each chunk of 128 terms costs a round
// trip (5 us), so the terms of a tile are cut among parts_x or parts_w blocks of a cluster of up to eight, and
// each adds up, in the blocks' order, the rows of the tile that fall to it: 6 x 812 x 128 in one block a
// tile took 38 us, cut 10.
template <typename T>
__global__ void __launch_bounds__(256)
small_grads_kernel(const Few p, int gx, int tiles_d, int parts_x, int parts_w)
{
    // 128 terms at a time, all their loads under way at once: the time is the latency of these rounds
    constexpr int K = kSmallTerms;
    __shared__ __align__(16) float a[K][36], b[K][36];   // [k][m], [k][n]
    __shared__ int counts[8];
    __shared__ bool use[1024];   // rows that are counted
    dep_wait();
    dep_release();
    const int tid = static_cast<int>(threadIdx.x);
    const bool dw = static_cast<int>(blockIdx.x) >= gx;
    const int parts = dw ? parts_w : parts_x;
    const int block = static_cast<int>(blockIdx.x) - (dw ? gx : 0), tile = block / parts, part = block - tile * parts;
    // blocks that fill the last cluster have rows past the end
    const int m0 = tile / tiles_d * 32, d0 = tile % tiles_d * 32;
    const int all = dw ? p.rows : static_cast<int>(p.vocab), ms = dw ? static_cast<int>(p.vocab) : p.rows;
    const int each = ((all + K - 1) / K + parts - 1) / parts * K, begin = part * each;
    const int terms = m0 < ms ? min(all, begin + each) : 0;
    const T* x = static_cast<const T*>(p.x);
    const T* w = static_cast<const T*>(p.w);
    const int tx = tid & 31, ty = tid >> 5;   // column; rows 4 ty ..
    const int vocab = static_cast<int>(p.vocab);
    // a chunk's operands, into registers: the next chunk's loads run under this one's products
    float la[K / 8], lb[K / 8];
    const auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < K / 8; ++i)
        {
            const int k = k0 + ty + 8 * i;
            if (dw)
            {
                // q as it lies: k = row, m = vocabulary
                la[i] = k < terms && m0 + tx < ms ? p.q[k * vocab + m0 + tx] : 0.0f;
                lb[i] = k < terms && d0 + tx < p.dim ? to_f32(x[k * p.ldx + d0 + tx]) : 0.0f;
            }
            else
            {
                // 32 rows of q, 128 columns of each
                const int m = m0 + ty + 8 * (i >> 2), c = k0 + tx + 32 * (i & 3);
                la[i] = m < ms && c < terms ? p.q[m * vocab + c] : 0.0f;
                lb[i] = k < terms && d0 + tx < p.dim ? to_f32(w[k * p.ldw + d0 + tx]) : 0.0f;
            }
        }
    };
    if (begin < terms) fetch(begin);
    int n = 0, bad = 0;
    for (int i = tid; i < p.rows; i += 256)
    {
        const int64_t t = p.targets[i];
        use[i] = counted(t, p.ignore, p.vocab);
        if (use[i]) ++n;
        else if (t != p.ignore) ++bad;
    }
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    if (blockIdx.x == 0 && __any_sync(0xFFFFFFFFu, bad != 0) && (tid & 31) == 0 && p.status != nullptr)
    {
        *p.status = VEDA_ERR_OUT_OF_RANGE;
    }
    if ((tid & 31) == 0) counts[tid >> 5] = n;
    __syncthreads();
    n = 0;
    for (int k = 0; k < 8; ++k) n += counts[k];
    const float coef = n > 0 ? (p.upstream != nullptr ? *p.upstream : 1.0f) / static_cast<float>(n) : 0.0f;

    // four slices of the terms, 64 threads each, a thread 4 x 4 of the tile
    const int slice = tid >> 6, om = (tid >> 3 & 7) * 4, on = (tid & 7) * 4;
    float acc[4][4] = {};
    for (int k0 = begin; k0 < terms; k0 += K)
    {
#pragma unroll
        for (int i = 0; i < K / 8; ++i)
        {
            const int k = k0 + ty + 8 * i;
            if (dw)
            {
                a[ty + 8 * i][tx] = la[i];
                // what an ignored row holds (NaN included) meets q = 0 as 0
                b[ty + 8 * i][tx] = k < terms && use[k] ? lb[i] : 0.0f;
            }
            else
            {
                a[tx + 32 * (i & 3)][ty + 8 * (i >> 2)] = la[i];
                b[ty + 8 * i][tx] = lb[i];
            }
        }
        __syncthreads();
        if (k0 + K < terms) fetch(k0 + K);
#pragma unroll 8
        for (int k = slice * (K / 4); k < (slice + 1) * (K / 4); ++k)
        {
            const float4 u = *reinterpret_cast<const float4*>(&a[k][om]);
            const float4 v = *reinterpret_cast<const float4*>(&b[k][on]);
            const float um[4] = {u.x, u.y, u.z, u.w}, vn[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
#pragma unroll
                for (int l = 0; l < 4; ++l) acc[i][l] = fmaf(um[i], vn[l], acc[i][l]);
            }
        }
        __syncthreads();
    }
    // the slices' sums meet in shared memory, added in order
    constexpr int kSum = 32 * 32;
    float* const sums = &a[0][0];   // [slice][32][32]
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
#pragma unroll
        for (int l = 0; l < 4; ++l) sums[(slice * 32 + om + i) * 32 + on + l] = acc[i][l];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        float* at = sums + (ty + 8 * i) * 32 + tx;
        at[0] = ((at[0] + at[kSum]) + at[2 * kSum]) + at[3 * kSum];
    }
    pair::cluster_arrive();   // the blocks' sums are there
    pair::cluster_wait();
    const int first = static_cast<int>(pair::cluster_rank()) - part, share = 32 / parts;
    for (int y = part * share + ty; y < (part + 1) * share; y += 8)
    {
        const int m = m0 + y;
        if (m >= ms || d0 + tx >= p.dim) continue;
        float v = 0.0f;
        for (int b = 0; b < parts; ++b)
        {
            float o;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(pair::peer_addr(sums + y * 32 + tx, first + b)));
            v += o;
        }
        v *= coef;
        if (!dw)
        {
            static_cast<T*>(p.dx)[m * p.lddx + d0 + tx] = from_f32<T>(v);
        }
        else if (p.dw_f32)
        {
            float* at = static_cast<float*>(p.dw) + m * p.lddw + d0 + tx;
            *at = p.dw_beta ? *at + v : v;
        }
        else
        {
            bf16* at = static_cast<bf16*>(p.dw) + m * p.lddw + d0 + tx;
            *at = __float2bfloat16_rn(p.dw_beta ? __bfloat162float(*at) + v : v);
        }
    }
    pair::cluster_sync();   // no block leaves while another may still read its sums
}

// ---- host ------------------------------------------------------------------------------------
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Where a call's scratch lies in its workspace (offsets in bytes, each a multiple of 256).
struct Layout
{
    int planes;
    int64_t ldp;          // pitch of the operand planes (elements)
    int64_t piece;        // columns of a piece of q (a multiple of 256)
    int64_t ld_acc;       // pitch of the fp32 dx sums
    int splits;           // of dx's sum over a piece
    int strip, slots;     // forward: tiles a strip, strips
    size_t scalars, done, part, row_scale, px, pw, parts, target_logit, q, acc, total;
};

// Tiles per strip: up to 8, by the number of tile times the busiest of `clusters` clusters runs;
// longer strips win ties (fewer partial pairs). 8192 rows x 151936: 8 (33 rounds of 8 against 257 of
// 1, within 3 %, an eighth of the pairs); a single row tile: 1 (9 rounds against 16 with 8).
int choose_strip(int num_m, int num_n, int clusters)
{
    int best = 1;
    int64_t best_time = INT64_MAX;
    for (int s = 1; s <= 8; s *= 2)
    {
        const int64_t units = static_cast<int64_t>((num_n + s - 1) / s) * num_m;
        const int64_t time = (units + clusters - 1) / clusters * s;
        if (time * 32 <= best_time * 33 || best_time == INT64_MAX)
        {
            best = s;
            best_time = std::min(time, best_time);
        }
    }
    return best;
}

// Columns of a tile: split products fold their accumulators under the next ones with narrow tiles only.
int tile_width(int dtype) { return dtype == VEDA_F32 ? 128 : 256; }

// Up to four rows of at most 2048 columns (a thread holds eight) go past the tensor cores. Against
// 151936 x 1024, forward / backward in runs: 1 row 53 / 128 us, 2 rows 53 / 151, 4 rows 67 / 213; the tensor tiles
// take 86 / 225 for 9 (8 rows on the CUDA cores: 101 / 359).
bool is_few(int64_t rows, int64_t dim) { return rows <= kFewRows && dim <= 2048; }

// Problems whose products the CUDA cores finish within the latency of the tensor-core path's launches, which
// is longer in fp32 and for odd widths (operands to lay out). Steps, here / tensor cores: bf16 16 x 1000 x 64
// 18.7 / 25.3 us, 8 x 4000 x 64 38 / 26, 5 x 600 x 1000 43 / 33, 128 x 512 x 64 25.7 / 25.6; fp32 128 x 512 x 64
// 23.3 / 34, 207 x 766 x 64 32.8 / 34.6, 500 x 500 x 64 42.5 / 36.5, 32 x 2000 x 256 39.0 / 37.8. (The tensor cores'
// times are of launches that overlapped; apart, as they are now, they take some 5 us more.)
bool is_small(int64_t rows, int64_t vocab, int64_t dim, int dtype)
{
    if (rows > 1024 || vocab > 4096 || dim > 1024)
    {
        return false;
    }
    const int64_t products = rows * vocab * dim;
    if (dtype == VEDA_BF16 && dim % 8 == 0)
    {
        return products <= (1 << 22) && vocab <= 1024 && vocab * dim <= (1 << 18);
    }
    return products <= (1 << 23);
}

Layout layout(int64_t rows, int64_t vocab, int64_t dim, bool pack_x, bool pack_w, int dtype, bool backward)
{
    Layout l{};
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += static_cast<size_t>(round_up(bytes, 256));
        return here;
    };
    if (is_few(rows, dim) || is_small(rows, vocab, dim, dtype))
    {
        l.done = take(4);
        l.parts = take(kFewBlocks * rows * 8);
        l.target_logit = take(rows * 4);
        l.ld_acc = round_up(dim, 4);
        l.acc = take(backward && is_few(rows, dim) ? kFewBlocks * rows * l.ld_acc * 4 : 0);
        l.q = take(backward && !is_few(rows, dim) ? rows * vocab * 4 : 0);
        l.total = at;
        return l;
    }
    l.planes = dtype == VEDA_F32 ? 2 : 1;
    l.ldp = round_up(dim, 8);
    l.scalars = take(sizeof(Scalars));
    l.done = take(4);
    l.part = take(2 * kMaxBlocks * 4);
    l.row_scale = take(!backward && dtype == VEDA_F32 ? rows * 4 : 0);
    l.px = take(pack_x ? l.planes * rows * l.ldp * 2 : 0);
    l.pw = take(pack_w ? l.planes * vocab * l.ldp * 2 : 0);
    const int tn = tile_width(dtype), num_n = static_cast<int>((vocab + tn - 1) / tn), num_m = static_cast<int>((rows + 255) / 256);
    if (!backward)
    {
        // at most 74 clusters on a B200; fewer (reserved SMs) only change which strip is best
        l.strip = choose_strip(num_m, num_n, 74);
        l.slots = (num_n + l.strip - 1) / l.strip;
        l.parts = take(static_cast<int64_t>(l.slots) * 2 * rows * 8);
        l.target_logit = take(rows * 4);
    }
    else
    {
        // Two pieces of q of about 64 MB: one is written while the other is read, mostly from L2, and
        // the launches are long enough for their tails not to count. Backward of 8192 x 151936 x 1024
        // with pieces of 8 / 16 / 32 / 64 / 128 MB: 13.4 / 7.71 / 6.42 / 6.06 / 6.27 ms.
        const int64_t fit = (int64_t{64} << 20) / (rows * 2 * l.planes) / 256 * 256;
        l.piece = std::min(round_up(vocab, 256), std::max<int64_t>(256, fit));
        l.q = take(2 * l.planes * rows * l.piece * 2);
        // Where dx has fewer tiles than the GPU has CTA pairs, its sums over a piece are cut into splits of
        // at least 8 k-blocks, each kept apart: one cluster summing 100000 columns for 16 rows of 768 took
        // 430 us by itself.
        const int64_t tiles = num_m * ((dim + tn - 1) / tn), kbs = (std::min(l.piece, vocab) + 63) / 64;
        const int64_t want = std::min((74 + tiles - 1) / tiles, (kbs + 7) / 8);
        l.splits = static_cast<int>((kbs + (kbs + want - 1) / want - 1) / ((kbs + want - 1) / want));
        l.ld_acc = round_up(dim, 4);
        l.acc = take(l.splits * rows * l.ld_acc * 4);
    }
    l.total = at;
    return l;
}

// Shares of `tiles[k]` tiles of `cost[k]` k-blocks each among the clusters: the costlier kinds first,
// each filled up to a common level, then one more tile each to the least loaded. Dealt out in turn
// instead, the clusters with a dW tile (128 k-blocks at 8192 rows) had 240 k-blocks of a launch's 166
// on average.
void share(const int64_t (&tiles)[3], const int64_t (&cost)[3], int clusters, Shares& out)
{
    int64_t load[kMaxClusters] = {}, count[3][kMaxClusters] = {};
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return cost[a] > cost[b]; });
    for (const int k : order)
    {
        int64_t lo = 0, hi = 0;   // the highest level that all of kind k's tiles still cover
        for (int c = 0; c < clusters; ++c) hi = std::max(hi, load[c]);
        hi += tiles[k] * cost[k] + 1;
        const auto fits = [&](int64_t level) {
            int64_t n = 0;
            for (int c = 0; c < clusters; ++c) n += level > load[c] ? (level - load[c]) / cost[k] : 0;
            return n <= tiles[k];
        };
        while (hi - lo > 1)
        {
            const int64_t mid = (lo + hi) / 2;
            (fits(mid) ? lo : hi) = mid;
        }
        int64_t left = tiles[k];
        for (int c = 0; c < clusters; ++c)
        {
            const int64_t n = lo > load[c] ? (lo - load[c]) / cost[k] : 0;
            count[k][c] = n;
            load[c] += n * cost[k];
            left -= n;
        }
        for (; left > 0; --left)
        {
            const int c = static_cast<int>(std::min_element(load, load + clusters) - load);
            ++count[k][c];
            load[c] += cost[k];
        }
    }
    for (int k = 0; k < 3; ++k)
    {
        int64_t at = 0;
        for (int c = 0; c <= kMaxClusters; ++c)
        {
            out.first[k][c] = static_cast<int>(at);
            at += c < clusters ? count[k][c] : 0;
        }
    }
}

struct Call
{
    const void *x, *w;
    int64_t ldx, ldw, rows, vocab, dim;
    int dtype;
    bool pack_x, pack_w, backward;
    Layout l;
    char* ws;
    Scalars* scalars() const { return reinterpret_cast<Scalars*>(ws + l.scalars); }
};

bool needs_pack(const void* m, int64_t ld, int dtype) { return dtype == VEDA_F32 || !aligned16(m) || ld % 8 != 0; }

unsigned pack_blocks(int64_t rows)
{
    return static_cast<unsigned>(std::min<int64_t>((rows + 7) / 8, kMaxBlocks));
}

// fp32: the largest magnitudes. Then the scalars, then the operand planes where the operands cannot
// be read in place, and the operands' tensor maps.
int prepare(const Call& c, const int64_t* targets, int64_t ignore, const float* upstream, int* status,
            bool scalars, Params& p, cudaStream_t s)
{
    float *part = nullptr, *row_scale = nullptr;
    const unsigned gx = pack_blocks(c.rows), gw = pack_blocks(c.vocab);
    if (c.dtype == VEDA_F32)
    {
        part = reinterpret_cast<float*>(c.ws + c.l.part);
        if (!c.backward) row_scale = reinterpret_cast<float*>(c.ws + c.l.row_scale);
        const int rc = launch("veda_linear_cross_entropy", absmax_kernel, dim3(gx + gw), dim3(256), 0, s,
                              static_cast<const float*>(c.x), c.ldx, c.rows, static_cast<const float*>(c.w), c.ldw,
                              c.vocab, c.dim, targets, ignore, static_cast<int>(gx), part, row_scale);
        if (rc != VEDA_OK) return rc;
    }
    const void *px = c.x, *pw = c.w;
    int64_t ldx = c.ldx, ldw = c.ldw;
    if (scalars || part != nullptr || c.pack_x || c.pack_w)
    {
        auto* ox = reinterpret_cast<uint16_t*>(c.ws + c.l.px);
        auto* ow = reinterpret_cast<uint16_t*>(c.ws + c.l.pw);
        const int64_t es = static_cast<int64_t>(dtype_size(c.dtype));
        const auto blocks = [&](int64_t n) {
            return static_cast<int>(std::min<int64_t>((n * (c.l.ldp / 8) + 255) / 256, 8ll * sm_count()));
        };
        const auto vec = [&](const void* m, int64_t ld) { return aligned16(m) && ld * es % 16 == 0; };
        const int bx = c.pack_x ? blocks(c.rows) : 0, bw = c.pack_w ? blocks(c.vocab) : 0;
        const auto go = [&](auto* x, auto* w, auto kernel) {
            return launch("veda_linear_cross_entropy (operands)", kernel, dim3(bx + bw + 1), dim3(256), 0, s, x, c.ldx,
                          c.rows, w, c.ldw, c.vocab, c.dim, targets, ignore, c.backward, vec(c.x, c.ldx), vec(c.w, c.ldw),
                          bx, bw, ox, ow, c.l.ldp, static_cast<const float*>(part), static_cast<int>(gx),
                          row_scale != nullptr ? 0 : static_cast<int>(gx), static_cast<int>(gw),
                          static_cast<const float*>(row_scale), upstream, c.scalars(), status);
        };
        const int rc = c.dtype == VEDA_F32
                           ? go(static_cast<const float*>(c.x), static_cast<const float*>(c.w), pack_kernel<float>)
                           : go(static_cast<const bf16*>(c.x), static_cast<const bf16*>(c.w), pack_kernel<bf16>);
        if (rc != VEDA_OK) return rc;
        if (c.pack_x)
        {
            px = ox;
            ldx = c.l.ldp;
        }
        if (c.pack_w)
        {
            pw = ow;
            ldw = c.l.ldp;
        }
    }
    const bool bf = c.dtype == VEDA_BF16;
    if (!pair::make_map3(&p.x, px, 2, bf, c.dim, c.rows, c.l.planes, ldx, c.rows * ldx, 64, bf ? 128 : 64) ||
        !pair::make_map3(&p.w, pw, 2, bf, c.dim, c.vocab, c.l.planes, ldw, c.vocab * ldw, 64, bf ? 128 : 64) ||
        (c.backward &&
         (!pair::make_map3(&p.x_mn, px, 2, bf, c.dim, c.rows, c.l.planes, ldx, c.rows * ldx, 64, 64) ||
          !pair::make_map3(&p.w_mn, pw, 2, bf, c.dim, c.vocab, c.l.planes, ldw, c.vocab * ldw, 64, 64))))
    {
        return fail(VEDA_ERR_CUDA, "veda_linear_cross_entropy: tensor map creation failed");
    }
    p.rows = static_cast<int>(c.rows);
    p.vocab = static_cast<int>(c.vocab);
    p.dim = static_cast<int>(c.dim);
    p.split = !bf;
    p.is_bf16 = bf;
    p.num_m = static_cast<int>((c.rows + 255) / 256);
    const int tn = tile_width(c.dtype);
    p.num_d = static_cast<int>((c.dim + tn - 1) / tn);
    p.by_m = pair::Divisor(static_cast<uint32_t>(p.num_m));
    p.by_d = pair::Divisor(static_cast<uint32_t>(p.num_d));
    p.scalars = c.scalars();
    p.row_scale = row_scale;
    p.targets = targets;
    p.ignore = ignore;
    p.status = device_status_ptr();
    return VEDA_OK;
}

// Common checks; fills c and its layout.
int check(Call& c, void* workspace, size_t bytes, bool backward, const char* name)
{
    c.backward = backward;
    c.pack_x = backward || needs_pack(c.x, c.ldx, c.dtype);
    c.pack_w = needs_pack(c.w, c.ldw, c.dtype);
    c.l = layout(c.rows, c.vocab, c.dim, c.pack_x, c.pack_w, c.dtype, backward);
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 || bytes < c.l.total)
    {
        return fail(VEDA_ERR_INVALID_ARGUMENT,
                    std::string(name) + ": workspace too small or not 256-byte aligned (see "
                                        "veda_linear_cross_entropy_workspace; a base that is not 16-byte aligned "
                                        "needs the size of a pitch that is no multiple of 8)");
    }
    c.ws = static_cast<char*>(workspace);
    return VEDA_OK;
}

// Elements of a row that can be accessed at a time: 8 (of fp32 by 16 bytes twice), 4, 2 or 1.
int grain(const void* base, int64_t ld, int dtype)
{
    const int64_t size = dtype == VEDA_BF16 ? 2 : 4;
    for (int64_t g = 8; g > 1; g /= 2)
    {
        const int64_t bytes = std::min<int64_t>(16, g * size);
        if (reinterpret_cast<uintptr_t>(base) % bytes == 0 && ld * size % bytes == 0) return static_cast<int>(g);
    }
    return 1;
}

// ---- few rows, host -----------------------------------------------------------------------------
Few few_params(const Call& c, const int64_t* targets, int64_t ignore, int* status)
{
    Few p{};
    p.x = c.x;
    p.w = c.w;
    p.ldx = c.ldx;
    p.ldw = c.ldw;
    p.rows = static_cast<int>(c.rows);
    p.dim = static_cast<int>(c.dim);
    p.padded = static_cast<int>(round_up(c.dim, 256));
    p.vocab = c.vocab;
    p.targets = targets;
    p.ignore = ignore;
    p.grain = grain(c.w, c.ldw, c.dtype);
    while (c.dim % p.grain != 0) p.grain /= 2;
    p.parts = reinterpret_cast<float2*>(c.ws + c.l.parts);
    p.target_logit = reinterpret_cast<float*>(c.ws + c.l.target_logit);
    p.acc = reinterpret_cast<float*>(c.ws + c.l.acc);
    p.ld_acc = c.l.ld_acc;
    p.q = reinterpret_cast<float*>(c.ws + c.l.q);
    p.done = reinterpret_cast<unsigned*>(c.ws + c.l.done);
    p.status = status;
    return p;
}

// Opts a kernel into `bytes` of dynamic shared memory on the current device.
template <typename K>
bool allow_smem(K kernel, int bytes)
{
    if (bytes <= 48 * 1024)
    {
        return true;
    }
    const bool ok = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
    cudaGetLastError();
    return ok;
}

// Blocks of a row group: what the SMs hold at once over all groups, or fewer where there are fewer pieces of
// the vocabulary.
int few_blocks(int64_t vocab, int piece, int per_sm, int groups)
{
    const int64_t room = std::max(1, per_sm * sm_count() / groups);
    return static_cast<int>(std::min<int64_t>({(vocab + piece - 1) / piece, room, kFewBlocks}));
}

template <typename T, int R, bool Q>
int launch_few_fwd(const Few& p, int* blocks, cudaStream_t s)
{
    const int groups = (p.rows + R - 1) / R;
    *blocks = few_blocks(p.vocab, 4 * kFewWarps, few_fwd_per_sm(R), groups);
    const int smem = R * p.padded * 4;
    const auto kernel = p.grain == 8   ? few_fwd_kernel<T, R, 8, Q>
                        : p.grain == 4 ? few_fwd_kernel<T, R, 4, Q>
                        : p.grain == 2 ? few_fwd_kernel<T, R, 2, Q>
                                       : few_fwd_kernel<T, R, 1, Q>;
    if (!allow_smem(kernel, smem))
    {
        return fail(VEDA_ERR_CUDA, "veda_linear_cross_entropy: shared memory");
    }
    return launch("veda_linear_cross_entropy", kernel, dim3(*blocks, groups), dim3(kFewThreads), smem, s, p);
}

template <typename T, int R>
int launch_few_bwd(Few p, int* blocks, cudaStream_t s)
{
    // 32 vocabulary rows at a time, fewer where two sets of them would pass an SM's shared memory
    const int room = 220 * 1024 / kFewBwdPerSm - 2048 - (R * p.padded + 32 * R) * 4;
    p.chunk = 32;
    while (p.chunk > 4 && 2 * p.chunk * p.padded * static_cast<int>(sizeof(T)) > room) p.chunk /= 2;
    *blocks = few_blocks(p.vocab, p.chunk, kFewBwdPerSm, 1);
    const int smem = (R * p.padded + 32 * R) * 4 + 2 * p.chunk * p.padded * static_cast<int>(sizeof(T));
    if (!allow_smem(few_bwd_kernel<T, R>, smem))
    {
        return fail(VEDA_ERR_CUDA, "veda_linear_cross_entropy_bwd: shared memory");
    }
    return launch("veda_linear_cross_entropy_bwd", few_bwd_kernel<T, R>, dim3(*blocks), dim3(kFewThreads), smem, s, p);
}

// As launch(), in clusters of `cluster` blocks.
template <typename... Params, typename... Args>
int launch_clusters(const char* what, void (*kernel)(Params...), int blocks, int threads, int cluster, cudaStream_t s,
                    Args&&... args)
{
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attrs[0].val.clusterDim.y = 1;
    attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.stream = s;
    cfg.attrs = attrs;
    cfg.numAttrs = overlapped_launches() ? 2 : 1;
    count_launch();
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
    if (err != cudaSuccess)
    {
        cudaGetLastError();
        return fail(VEDA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(err));
    }
    return check_launch(what);
}

int launch_merge(const float2* parts, int slots, int64_t rows, int64_t vocab, const int64_t* targets, int64_t ignore,
                 const float* target_logit, float* row_loss, float* lse, float* loss, unsigned* done, int* status,
                 cudaStream_t s)
{
    // 32 rows a block reads whole lines of pairs; fewer where the rows would not fill the GPU's SMs
    int width = 32;
    while (width > 1 && (rows + width - 1) / width < sm_count()) width /= 2;
    return launch("veda_linear_cross_entropy_fwd (merge)", merge_kernel,
                  dim3(static_cast<unsigned>((rows + width - 1) / width)), dim3(256), 0, s, parts, slots, rows, vocab,
                  width, targets, ignore, target_logit, row_loss, lse, loss, done, status);
}

template <typename T>
int few_fwd(const Call& c, const int64_t* targets, int64_t ignore, float* row_loss, float* lse, float* loss, int* status,
            cudaStream_t s)
{
    const Few p = few_params(c, targets, ignore, status);
    int blocks = 0;
    const int rc = p.rows == 1   ? launch_few_fwd<T, 1, false>(p, &blocks, s)
                   : p.rows == 2 ? launch_few_fwd<T, 2, false>(p, &blocks, s)
                                 : launch_few_fwd<T, 4, false>(p, &blocks, s);
    if (rc != VEDA_OK) return rc;
    return launch_merge(p.parts, blocks, c.rows, c.vocab, targets, ignore, p.target_logit, row_loss, lse, loss, p.done,
                        status, s);
}

template <typename T>
int small_bwd(const Call& c, const int64_t* targets, int64_t ignore, const float* lse, const float* upstream, void* dx,
              int64_t lddx, void* dw, int64_t lddw, int dtype_dw, bool beta, int* status, cudaStream_t s)
{
    Few p = few_params(c, targets, ignore, status);
    p.lse = lse;
    p.upstream = upstream;
    p.dx = dx;
    p.lddx = lddx;
    p.dw = dw;
    p.lddw = lddw;
    p.dw_f32 = dtype_dw == VEDA_F32;
    p.dw_beta = beta;
    int blocks = 0;
    const int rc = launch_few_fwd<T, 4, true>(p, &blocks, s);
    if (rc != VEDA_OK) return rc;
    const int tiles_d = (p.dim + 31) / 32;
    const auto parts_of = [](int64_t terms) {
        int k = 1;
        while (k < 8 && k * kSmallTerms < terms) k *= 2;
        return k;
    };
    const int parts_x = parts_of(c.vocab), parts_w = parts_of(p.rows);
    const int cluster = std::max(dx != nullptr ? parts_x : 1, dw != nullptr ? parts_w : 1);
    const auto whole = [&](int64_t blocks) { return static_cast<int>(round_up(blocks, cluster)); };
    const int gx = dx != nullptr ? whole((p.rows + 31) / 32 * tiles_d * parts_x) : 0;
    const int gw = dw != nullptr ? whole((c.vocab + 31) / 32 * tiles_d * parts_w) : 0;
    if (gx + gw == 0) return VEDA_OK;
    return launch_clusters("veda_linear_cross_entropy_bwd", small_grads_kernel<T>, gx + gw, 256, cluster, s, p, gx, tiles_d, parts_x, parts_w);
}

template <typename T>
int few_bwd(const Call& c, const int64_t* targets, int64_t ignore, const float* lse, const float* upstream, void* dx,
            int64_t lddx, void* dw, int64_t lddw, int dtype_dw, bool beta, int* status, cudaStream_t s)
{
    Few p = few_params(c, targets, ignore, status);
    p.lse = lse;
    p.upstream = upstream;
    p.dw = dw;
    p.lddw = lddw;
    p.dw_f32 = dtype_dw == VEDA_F32;
    p.dw_beta = beta;
    // groups of 4 or 2 have to end with the row; where groups of 8 do not, the last columns are written singly
    p.dw_grain = grain(dw, lddw, dtype_dw);
    while (p.dw_grain < 8 && c.dim % p.dw_grain != 0) p.dw_grain /= 2;
    if (dx == nullptr) p.acc = nullptr;
    int blocks = 0;
    int rc = p.rows == 1   ? launch_few_bwd<T, 1>(p, &blocks, s)
             : p.rows == 2 ? launch_few_bwd<T, 2>(p, &blocks, s)
                           : launch_few_bwd<T, 4>(p, &blocks, s);
    if (rc != VEDA_OK || dx == nullptr) return rc;
    return launch("veda_linear_cross_entropy_bwd (dx)", few_dx_kernel<T>, dim3((p.dim + 31) / 32, p.rows), dim3(256), 0, s,
                  p, blocks, static_cast<T*>(dx), lddx);
}

constexpr int64_t kLimit = (1ll << 31) - 512;   // tile coordinates are 32-bit

} // namespace lce
} // namespace veda::cuda

using namespace veda::cuda;

extern "C" size_t veda_linear_cross_entropy_workspace(int64_t rows, int64_t vocab, int64_t dim, int64_t ldx,
                                                      int64_t ldw, int dtype, int backward)
{
    if (rows <= 0 || vocab <= 0 || dim <= 0 || rows > lce::kLimit || vocab > lce::kLimit || dim > lce::kLimit ||
        !valid_dtype(dtype))
    {
        return 0;
    }
    return lce::layout(rows, vocab, dim, backward != 0 || dtype == VEDA_F32 || ldx % 8 != 0, dtype == VEDA_F32 || ldw % 8 != 0, dtype,
                       backward != 0)
        .total;
}

extern "C" int veda_linear_cross_entropy_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                             const int64_t* targets, int64_t ignore_index, float* row_loss, float* lse,
                                             float* loss, int64_t rows, int64_t vocab, int64_t dim, void* workspace,
                                             size_t workspace_bytes, int* status, int dtype, veda_stream_t stream)
{
    VEDA_REQUIRE(valid_dtype(dtype), "unknown dtype");
    VEDA_REQUIRE(rows >= 0 && vocab > 0 && dim > 0, "bad shape");
    VEDA_REQUIRE(rows <= lce::kLimit && vocab <= lce::kLimit && dim <= lce::kLimit, "an extent does not fit 31 bits");
    VEDA_REQUIRE(ldx >= dim && ldw >= dim, "leading dimension smaller than dim");
    if (rows == 0)
    {
        // nothing to average over: 0, as for a batch of ignored rows
        if (loss != nullptr && cudaMemsetAsync(loss, 0, sizeof(float), stream) != cudaSuccess)
        {
            return fail(VEDA_ERR_CUDA, "veda_linear_cross_entropy_fwd: clearing the loss failed");
        }
        return VEDA_OK;
    }
    VEDA_REQUIRE(x != nullptr && w != nullptr && targets != nullptr && row_loss != nullptr, "null pointer");
    lce::Call c{x, w, ldx, ldw, rows, vocab, dim, dtype};
    int rc = lce::check(c, workspace, workspace_bytes, false, "veda_linear_cross_entropy_fwd");
    if (rc != VEDA_OK) return rc;
    if (lce::is_few(rows, dim) || lce::is_small(rows, vocab, dim, dtype))
    {
        return dtype == VEDA_BF16
                   ? lce::few_fwd<bf16>(c, targets, ignore_index, row_loss, lse, loss, status, stream)
                   : lce::few_fwd<float>(c, targets, ignore_index, row_loss, lse, loss, status, stream);
    }
    const bool split = dtype == VEDA_F32;
    const int clusters = split ? pair::clusters_available<lce::StatsWork<128>, 4, true>()
                               : pair::clusters_available<lce::StatsWork<256>, 4, false>();
    if (clusters < 1)
    {
        return pair::none_available("veda_linear_cross_entropy_fwd", clusters);
    }
    lce::Params p{};
    rc = lce::prepare(c, targets, ignore_index, nullptr, nullptr, false, p, stream);
    if (rc != VEDA_OK) return rc;
    p.num_n = static_cast<int>((vocab + lce::tile_width(dtype) - 1) / lce::tile_width(dtype));
    while ((1 << p.strip_log2) < c.l.strip) ++p.strip_log2;
    p.parts = reinterpret_cast<float2*>(c.ws + c.l.parts);
    p.target_logit = reinterpret_cast<float*>(c.ws + c.l.target_logit);
    p.done = reinterpret_cast<unsigned*>(c.ws + c.l.done);
    const int64_t units = static_cast<int64_t>(c.l.slots) * p.num_m;
    VEDA_REQUIRE(units <= lce::kLimit, "too many tiles");
    const int grid = static_cast<int>(std::min<int64_t>(units, clusters));
    rc = split ? pair::launch_pair<lce::StatsWork<128>, 4, true>("veda_linear_cross_entropy_fwd", p, grid, false, stream)
               : pair::launch_pair<lce::StatsWork<256>, 4, false>("veda_linear_cross_entropy_fwd", p, grid, false, stream);
    if (rc != VEDA_OK) return rc;
    return lce::launch_merge(p.parts, c.l.slots, rows, vocab, targets, ignore_index, p.target_logit, row_loss, lse, loss,
                             p.done, status, stream);
}

extern "C" int veda_linear_cross_entropy_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                             const int64_t* targets, int64_t ignore_index, const float* lse,
                                             const float* upstream, void* dx, int64_t lddx, void* dw, int64_t lddw,
                                             int dtype_dw, float beta_dw, int64_t rows, int64_t vocab, int64_t dim,
                                             void* workspace, size_t workspace_bytes, int* status, int dtype,
                                             veda_stream_t stream)
{
    VEDA_REQUIRE(valid_dtype(dtype) && valid_dtype(dtype_dw), "unknown dtype");
    VEDA_REQUIRE(dtype == VEDA_BF16 || dtype_dw == VEDA_F32, "fp32 operands have an fp32 weight gradient");
    VEDA_REQUIRE(rows >= 0 && vocab > 0 && dim > 0, "bad shape");
    VEDA_REQUIRE(rows <= lce::kLimit && vocab <= lce::kLimit && dim <= lce::kLimit, "an extent does not fit 31 bits");
    VEDA_REQUIRE(ldx >= dim && ldw >= dim, "leading dimension smaller than dim");
    VEDA_REQUIRE((dx == nullptr || lddx >= dim) && (dw == nullptr || lddw >= dim),
                 "gradient leading dimension smaller than dim");
    VEDA_REQUIRE(beta_dw == 0.0f || beta_dw == 1.0f, "beta_dw must be 0 (overwrite) or 1 (accumulate)");
    if (rows == 0)
    {
        if (dw != nullptr && beta_dw == 0.0f &&
            cudaMemset2DAsync(dw, lddw * dtype_size(dtype_dw), 0, dim * dtype_size(dtype_dw), vocab, stream) != cudaSuccess)
        {
            return fail(VEDA_ERR_CUDA, "veda_linear_cross_entropy_bwd: clearing dw failed");
        }
        return VEDA_OK;
    }
    VEDA_REQUIRE(x != nullptr && w != nullptr && targets != nullptr && lse != nullptr, "null pointer");
    if (dx == nullptr && dw == nullptr)
    {
        return VEDA_OK;
    }
    lce::Call c{x, w, ldx, ldw, rows, vocab, dim, dtype};
    int rc = lce::check(c, workspace, workspace_bytes, true, "veda_linear_cross_entropy_bwd");
    if (rc != VEDA_OK) return rc;
    if (lce::is_few(rows, dim))
    {
        return dtype == VEDA_BF16 ? lce::few_bwd<bf16>(c, targets, ignore_index, lse, upstream, dx, lddx, dw, lddw,
                                                       dtype_dw, beta_dw != 0.0f, status, stream)
                                  : lce::few_bwd<float>(c, targets, ignore_index, lse, upstream, dx, lddx, dw, lddw,
                                                        dtype_dw, beta_dw != 0.0f, status, stream);
    }
    if (lce::is_small(rows, vocab, dim, dtype))
    {
        return dtype == VEDA_BF16 ? lce::small_bwd<bf16>(c, targets, ignore_index, lse, upstream, dx, lddx, dw, lddw,
                                                         dtype_dw, beta_dw != 0.0f, status, stream)
                                  : lce::small_bwd<float>(c, targets, ignore_index, lse, upstream, dx, lddx, dw, lddw,
                                                          dtype_dw, beta_dw != 0.0f, status, stream);
    }
    const bool split = dtype == VEDA_F32;
    const int clusters = std::min(lce::kMaxClusters, split ? pair::clusters_available<lce::GradWork<128>, 8, true>()
                                                           : pair::clusters_available<lce::GradWork<256>, 8, false>());
    if (clusters < 1)
    {
        return pair::none_available("veda_linear_cross_entropy_bwd", clusters);
    }
    lce::Params p{};
    rc = lce::prepare(c, targets, ignore_index, upstream, status, true, p, stream);
    if (rc != VEDA_OK) return rc;
    const int64_t piece = c.l.piece, plane = rows * piece;
    const bool bf = dtype == VEDA_BF16;
    CUtensorMap q_load[2], q_mn[2], q_store[2];
    bool ok = true;
    for (int b = 0; b < 2; ++b)
    {
        char* q = c.ws + c.l.q + static_cast<size_t>(b) * c.l.planes * plane * 2;
        ok = ok && pair::make_map3(&q_load[b], q, 2, bf, piece, rows, c.l.planes, piece, plane, 64, bf ? 128 : 64) &&
             pair::make_map3(&q_mn[b], q, 2, bf, piece, rows, c.l.planes, piece, plane, 64, 64) &&
             pair::make_map3(&q_store[b], q, 2, bf, piece, rows, c.l.planes, piece, plane, 64, 32);
    }
    float* acc = reinterpret_cast<float*>(c.ws + c.l.acc);
    ok = ok && pair::make_map3(&p.dx, acc, 4, false, dim, rows, c.l.splits, c.l.ld_acc, rows * c.l.ld_acc, 32, 32);
    p.dw_f32 = dtype_dw == VEDA_F32;
    p.dw_beta = beta_dw != 0.0f;
    p.dw_ptr = dw;
    p.lddw = lddw;
    if (dw != nullptr)
    {
        const int es = p.dw_f32 ? 4 : 2;
        const bool fits = aligned16(dw) && lddw * es % 16 == 0 && !(p.dw_beta && !p.dw_f32);
        if (fits && pair::make_map3(&p.dw, dw, es, !p.dw_f32, dim, vocab, 1, lddw, vocab * lddw, 128 / es, 32))
        {
            p.dw_mode = p.dw_beta ? 2 : 1;
        }
    }
    if (!ok)
    {
        return fail(VEDA_ERR_CUDA, "veda_linear_cross_entropy_bwd: tensor map creation failed");
    }
    p.lse = lse;
    p.q_in = q_load[0];
    p.q_mn = q_mn[0];
    // launch c: q of piece c, and the products of piece c - 1
    const int64_t pieces = (vocab + piece - 1) / piece;
    for (int64_t k = 0; k <= pieces; ++k)
    {
        int64_t tiles[3] = {};
        if (k < pieces)
        {
            p.v0 = static_cast<int>(k * piece);
            // q is written up to the next multiple of 256 columns, zero past the vocabulary
            tiles[lce::kQ] = (std::min(piece, vocab - k * piece) + 255) / 256 * (256 / lce::tile_width(dtype)) * p.num_m;
            p.q_out = q_store[k & 1];
        }
        if (k > 0)
        {
            p.g0 = static_cast<int>((k - 1) * piece);
            p.gcols = static_cast<int>(std::min(piece, vocab - (k - 1) * piece));
            p.q_in = q_load[(k - 1) & 1];
            p.q_mn = q_mn[(k - 1) & 1];
            tiles[lce::kDw] = dw != nullptr ? static_cast<int64_t>((p.gcols + 255) / 256) * p.num_d : 0;
            // a short last piece may fill fewer splits; all were stored with the first
            const int kbs = (p.gcols + pair::kBK - 1) / pair::kBK;
            p.dx_tiles = p.num_m * p.num_d;
            p.by_dx = pair::Divisor(static_cast<uint32_t>(p.dx_tiles));
            p.dx_kbs = (kbs + c.l.splits - 1) / c.l.splits;
            tiles[lce::kDx] =
                dx != nullptr ? static_cast<int64_t>((kbs + p.dx_kbs - 1) / p.dx_kbs) * p.dx_tiles : 0;
            p.dx_add = k > 1;
        }
        const int64_t units = tiles[0] + tiles[1] + tiles[2];
        VEDA_REQUIRE(units <= lce::kLimit, "too many tiles");
        const int grid = static_cast<int>(std::min<int64_t>(units, clusters));
        // k-blocks a tile, and what its epilogue adds
        const int64_t cost[3] = {(rows + 63) / 64 + 4, p.dx_kbs + 2, (dim + 63) / 64 + 2};
        lce::share(tiles, cost, grid, p.shares);
        rc = split ? pair::launch_pair<lce::GradWork<128>, 8, true>("veda_linear_cross_entropy_bwd", p, grid, k > 0, stream)
                   : pair::launch_pair<lce::GradWork<256>, 8, false>("veda_linear_cross_entropy_bwd", p, grid, k > 0, stream);
        if (rc != VEDA_OK) return rc;
    }
    if (dx == nullptr)
    {
        return VEDA_OK;
    }
    const lce::Scalars* scalars = c.scalars();
    const auto finish = [&](auto* out, auto one, auto several) {
        if (c.l.splits > 8 && rows * dim < 65536)
        {
            return launch("veda_linear_cross_entropy_bwd (dx)", several,
                          dim3(static_cast<unsigned>((dim + 31) / 32), static_cast<unsigned>(rows)), dim3(256), 0, stream,
                          static_cast<const float*>(acc), c.l.ld_acc, c.l.splits, out, lddx, rows, dim, scalars);
        }
        const int64_t es = static_cast<int64_t>(dtype_size(dtype));
        const bool vec = aligned16(dx) && lddx * es % 16 == 0;
        const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((rows * ((dim + 7) / 8) + 255) / 256, 8ll * sm_count()));
        return launch("veda_linear_cross_entropy_bwd (dx)", one, dim3(blocks), dim3(256), 0, stream,
                      static_cast<const float*>(acc), c.l.ld_acc, c.l.splits, out, lddx, rows, dim, vec, scalars);
    };
    return bf ? finish(static_cast<bf16*>(dx), lce::finish_dx_kernel<bf16>, lce::finish_splits_kernel<bf16>)
              : finish(static_cast<float*>(dx), lce::finish_dx_kernel<float>, lce::finish_splits_kernel<float>);
}
