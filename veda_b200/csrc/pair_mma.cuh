// A persistent CTA-pair tensor-core kernel over a list of 256 x 256 output tiles (or 256 x 128, where
// there are too few tiles for all SMs and a tile's latency counts), with the list and the epilogue
// supplied by a Work type: the mainloop of the loss head (linear_ce.cu) and of the
// Newton-Schulz products (newton_schulz.cu).
//
// A cluster of two CTAs computes a tile with tcgen05.mma.cta_group::2 (M 256, N 256, K 16; 16-bit
// operands, fp32 accumulators in TMEM). Each CTA stages its own 128 rows of A and 128 columns of B
// (32 KB per 64-deep k-block, five or six stages), the even CTA issues the products, two 256-column
// accumulators alternate so that a tile's epilogue runs under the next tile's products. Operands are
// read through 3-D tensor maps (column, row, plane): K-major pieces as one 64 x 128 box, MN-major
// ones as two 64 x 64 boxes. Loads carry no multicast. Every wait is bounded (tc::mbar_wait).
// Timestamps of the roles set the rest: a tile's coordinates are worked out while the tile before it
// is in flight (its divisions held the product thread up by 600 to 2000 cycles a tile, against 8192
// of products for k = 1024), and a k-block costs the loading thread additions only.
//
// SPLIT: operands are pairs of fp16 planes, value = hi + lo, and a product is hi lo + lo hi + hi hi.
// The tensor core truncates as it adds into its accumulator, always towards zero: sums of 10000 terms came out 3e-5
// short. So the small products go first, and every CHAIN k-blocks the accumulator is folded into a running sum kept
// in another part of TMEM, rounded to nearest: where all terms have one sign, 1.5e-6 of the sum are missing with
// chains of 4 k-blocks, whatever its length, and 3.2e-6 with chains of 8. With
// TN = 128 two accumulators and the sum fit, and a fold runs under the next chain's products; with TN = 256
// the accumulator has no second buffer then, and the products wait for it.
//
// Work provides
//   int TN, CHAIN                      columns of a tile; SPLIT: k-blocks between folds
//   struct Params                      the kernel's argument (tensor maps, pointers, sizes, status)
//   struct Tile { bool skip; int kbs; uint32_t idesc; bool a_mn, b_mn; ... }
//   bool tile(p, cid, clusters, i, t)  the i-th tile of cluster cid; false at the end of its list
//   void operands(p, t, rank, a, b)    where the operand pieces of CTA `rank` lie at k = 0
//   void prefetch(p)                   fetches the tensor maps of the operands
//   void ready(p, t, abort)            by one thread, before the tile's operands are loaded
//   void before(p, t, state, ...)      per epilogue warp, while the tile's products run
//   void epilogue(p, t, state, ...)    one warp's 32 rows x COLS columns of the finished tile
//   void after(p, t, lane)             per epilogue warp, the accumulator handed back
// All roles walk the same list, so tile() must depend on its arguments and on Params alone.
#pragma once

#include "tc_common.cuh"

namespace veda::cuda::pair
{

constexpr int kTile = 256;   // tile rows of a CTA pair, and columns unless the Work has TN = 128
constexpr int kBK = 64;      // k-block: 64 16-bit values, one 128-byte swizzle row

template <int EPI_WARPS_, int TN = kTile>
struct Cfg
{
    static constexpr int EPI_WARPS = EPI_WARPS_;   // 4, or 8 with half the columns each
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int STAGES = EPI_WARPS == 8 && TN == kTile ? 5 : 6;
    static constexpr int A_BYTES = 128 * kBK * 2;      // one CTA's half of the operands' k-block
    static constexpr int B_BYTES = TN / 2 * kBK * 2;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGE_TILE = 32 * 128;     // epilogue staging: 32 rows x 128 bytes
    static constexpr int STAGING = EPI_WARPS * 2 * STAGE_TILE;
    static constexpr int SMEM = STAGES * STAGE + STAGING + 1024 + 256;
};

// An operand piece at k = 0, 128 rows of A or TN / 2 of B by 64 terms: k runs along x (K-major, one box
// 64 x 128; with TN = 128 one or two of 64 x 64, one below the other) or along y (MN-major, boxes
// 64 x 64 side by side). z is the hi plane, z + 1 the lo plane of split operands.
struct Piece
{
    const CUtensorMap* map;
    int x, y, z;
};

// kind::f16 instruction descriptor: fp32 accumulators, A and B both bf16 or both fp16.
template <int TN = kTile>
__host__ __device__ constexpr uint32_t idesc(bool is_bf16, bool a_mn, bool b_mn)
{
    const uint32_t type = is_bf16 ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(TN >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

// n / d for 0 <= n < 2^31 by a multiplication: m = ceil(2^(31 + s) / d) with 2^s >= d.
struct Divisor
{
    uint32_t m = 0, s = 0, d = 1;
    Divisor() = default;
    __host__ explicit Divisor(uint32_t n) : d(n)
    {
        while ((1ull << s) < n) ++s;
        m = static_cast<uint32_t>(((1ull << (31 + s)) + n - 1) / n);
    }
    __device__ __forceinline__ int div(int n, int& rest) const
    {
        const int q = d == 1 ? n : static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> (31 + s));
        rest = n - q * static_cast<int>(d);
        return q;
    }
};

// One lane of the converged warp.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// shared::cluster address of a shared variable at the same place in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(tc::smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// A whole warp's bounded wait, converged afterwards (the elected lane issues for all, and tensor memory is read by
// whole warps); false once a wait of the CTA has given up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t phase, int* status, volatile int* abort)
{
    bool ok = tc::mbar_try_wait(tc::smem_u32(bar), phase);
    if (!ok)
    {
        tc::mbar_wait(bar, phase, status, abort);
        ok = *abort == 0;
    }
    return __all_sync(0xFFFFFFFFu, ok);
}
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void reduce_add_3d(const CUtensorMap* map, const void* src, int x, int y, int z)
{
    asm volatile(
        "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(tc::smem_u32(src)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void mma2(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(desc), "r"(accumulate));
}
__device__ __forceinline__ void commit2(uint64_t* bar)
{
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(tc::smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

// One warp's staging tiles (two of 32 rows x 128 bytes): buffer() waits until the bulk group that
// used the next one has read it and gives the tile; sent() counts the group just committed by lane 0.
struct Staging
{
    uint8_t* base;
    uint32_t count = 0;
    __device__ __forceinline__ uint8_t* buffer(int lane)
    {
        if (count >= 2)
        {
            if (lane == 0)
            {
                tc::bulk_wait_group_read<1>();
            }
            __syncwarp();
        }
        return base + (count & 1) * Cfg<4>::STAGE_TILE;
    }
    __device__ __forceinline__ void sent() { ++count; }
};

// SPLIT: adds the accumulator at `acc` (COLS columns) onto the running sum at `sum`, or starts it;
// the last fold leaves the total at `acc`, where the epilogue reads it.
template <int COLS>
__device__ __forceinline__ void fold(uint32_t acc, uint32_t sum, bool first, bool last)
{
#pragma unroll 1
    for (int c = 0; c < COLS; c += 32)
    {
        uint32_t a[32];
        tc::tmem_ld32(acc + static_cast<uint32_t>(c), a);
        if (!first)
        {
            uint32_t b[32];
            tc::tmem_ld32(sum + static_cast<uint32_t>(c), b);
#pragma unroll
            for (int j = 0; j < 32; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) + __uint_as_float(b[j]));
        }
        tc::tmem_st32((last ? acc : sum) + static_cast<uint32_t>(c), a);
    }
}

template <class Work, int EPI_WARPS, bool SPLIT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Cfg<EPI_WARPS, Work::TN>::THREADS, 1)
pair_kernel(const __grid_constant__ typename Work::Params p)
{
    using namespace tc;
    using C_ = Cfg<EPI_WARPS, Work::TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* sa = smem;
    constexpr int TN = Work::TN;
    constexpr bool TWO = !SPLIT || TN < kTile;   // two accumulators
    uint8_t* sb = smem + C_::STAGES * C_::A_BYTES;
    uint8_t* staging = sb + C_::STAGES * C_::B_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + C_::STAGING);
    uint64_t* empty = full + C_::STAGES;
    uint64_t* tfull = empty + C_::STAGES;
    uint64_t* tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);   // known to be the same in all lanes
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int cid = static_cast<int>(blockIdx.x >> 1);
    const int clusters = static_cast<int>(gridDim.x >> 1);

    if (threadIdx.x == 0)
    {
        *abort = 0;
        for (int s = 0; s < C_::STAGES; ++s)
        {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b)
        {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 2 * EPI_WARPS);   // the epilogue warps of both CTAs
        }
        mbar_fence_init();
    }
    if (warp == 1)
    {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    cluster_sync();   // both CTAs' barriers exist before any signal crosses
    fence_after();
    const uint32_t tmem = *tmem_slot;
    if (threadIdx.x == 0)
    {
        Work::prefetch(p);   // the maps are arguments: no need to wait for the kernels before
    }
    dep_wait();
    dep_release();

    typename Work::Tile t, next;
    bool more = Work::tile(p, cid, clusters, 0, t);
    int i = 0;
    if (warp == 0)
    {
        const bool leader = elect_one();
        int stage = 0;
        uint32_t phase = 0;
        while (more)
        {
            if (!t.skip)
            {
                if (leader)
                {
                    Work::ready(p, t, abort);
                }
                __syncwarp();
                Piece a, b;
                Work::operands(p, t, static_cast<int>(rank), a, b);
                const int adx = t.a_mn ? 0 : kBK, ady = t.a_mn ? kBK : 0;
                const int bdx = t.b_mn ? 0 : kBK, bdy = t.b_mn ? kBK : 0;
                auto load = [&](int kb, int za, int zb) {
                    if (!warp_wait(&empty[stage], phase ^ 1, p.status, abort))
                    {
                        return;   // nothing frees the stages any more
                    }
                    const uint32_t bar = peer_addr(&full[stage], 0);
                    uint8_t* ad = sa + stage * C_::A_BYTES;
                    uint8_t* bd = sb + stage * C_::B_BYTES;
                    const int ax = a.x + kb * adx, ay = a.y + kb * ady;
                    const int bx = b.x + kb * bdx, by = b.y + kb * bdy;
                    if (leader)
                    {
                        if (rank == 0)
                        {
                            mbar_expect_tx(&full[stage], 2 * C_::STAGE);   // both CTAs' halves
                        }
                        load_box(ad, a.map, bar, ax, ay, a.z + za);
                        if (t.a_mn) load_box(ad + C_::A_BYTES / 2, a.map, bar, ax + 64, ay, a.z + za);
                        else if (TN < kTile) load_box(ad + C_::A_BYTES / 2, a.map, bar, ax, ay + 64, a.z + za);
                        load_box(bd, b.map, bar, bx, by, b.z + zb);
                        if (TN == kTile && t.b_mn) load_box(bd + C_::B_BYTES / 2, b.map, bar, bx + 64, by, b.z + zb);
                    }
                    __syncwarp();
                    if (++stage == C_::STAGES)
                    {
                        stage = 0;
                        phase ^= 1;
                    }
                };
                if constexpr (!SPLIT)
                {
                    for (int kb = 0; kb < t.kbs; ++kb) load(kb, 0, 0);
                }
                else
                {
                    for (int k0 = 0; k0 < t.kbs; k0 += Work::CHAIN)
                    {
                        const int k1 = min(t.kbs, k0 + Work::CHAIN);
                        for (int kb = k0; kb < k1; ++kb) load(kb, 0, 1);
                        for (int kb = k0; kb < k1; ++kb) load(kb, 1, 0);
                        for (int kb = k0; kb < k1; ++kb) load(kb, 0, 0);
                    }
                }
            }
            more = Work::tile(p, cid, clusters, ++i, t);   // the ring is full of this tile's blocks
        }
        // The last release of every stage arrives before the CTA leaves: its signals cross CTAs on their own, and
        // the next kernel's barriers take these barriers' place.
        for (int s = 0; s < C_::STAGES; ++s)
        {
            warp_wait(&empty[stage], phase ^ 1, p.status, abort);
            if (++stage == C_::STAGES)
            {
                stage = 0;
                phase ^= 1;
            }
        }
    }
    else if (warp == 1 && rank == 0)
    {
        // The whole warp walks the tiles and works out the descriptors, in registers that it shares, and
        // one lane issues: under a branch for one thread a product took some 110 cycles to issue, and four
        // of them with their barriers more than the 512 that a k-block takes to multiply.
        const bool leader = elect_one();
        int stage = 0, it = 0;
        uint32_t phase = 0;
        while (more)
        {
            bool more_next = false;
            if (t.skip)
            {
                more_next = Work::tile(p, cid, clusters, ++i, next);
            }
            const uint32_t astep = (t.a_mn ? 2048 : 32) / 16, bstep = (t.b_mn ? 2048 : 32) / 16;   // 16 terms on
            const uint32_t albo = t.a_mn ? kBK * 128 : 16, blbo = t.b_mn ? kBK * 128 : 16;
            for (int k0 = 0; !t.skip && k0 < t.kbs; k0 += SPLIT ? Work::CHAIN : t.kbs)
            {
                const int blocks = SPLIT ? 3 * (min(t.kbs, k0 + Work::CHAIN) - k0) : t.kbs;
                const int buf = TWO ? it & 1 : 0;
                warp_wait(&tempty[buf], ((TWO ? it >> 1 : it) & 1) ^ 1, p.status, abort);
                fence_after();
                const uint32_t d = tmem + static_cast<uint32_t>(buf * TN);
                for (int kb = 0; kb < blocks; ++kb)
                {
                    if (!warp_wait(&full[stage], phase, p.status, abort))
                    {
                        break;
                    }
                    fence_after();
                    const uint64_t ad = smem_desc(smem_u32(sa + stage * C_::A_BYTES), albo, 1024);
                    const uint64_t bd = smem_desc(smem_u32(sb + stage * C_::B_BYTES), blbo, 1024);
                    if (leader)
                    {
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; ++kk)
                        {
                            mma2(d, ad + kk * astep, bd + kk * bstep, t.idesc, (kb > 0 || kk > 0) ? 1u : 0u);
                        }
                        commit2(&empty[stage]);
                    }
                    __syncwarp();
                    if (++stage == C_::STAGES)
                    {
                        stage = 0;
                        phase ^= 1;
                    }
                    if (kb == 0 && k0 == 0)
                    {
                        more_next = Work::tile(p, cid, clusters, ++i, next);   // under the products
                    }
                }
                if (leader) commit2(&tfull[buf]);
                __syncwarp();
                ++it;
            }
            t = next;
            more = more_next;
        }
    }
    else if (warp >= 2)
    {
        const int quarter = warp & 3;   // the TMEM lanes this warp may read
        constexpr int COLS = TN / (EPI_WARPS / 4);
        const int col0 = ((warp - 2) >> 2) * COLS;
        const int row0 = static_cast<int>(rank) * 128 + quarter * 32;   // within the tile
        const uint32_t release = peer_addr(&tempty[0], 0);
        Staging st{staging + (warp - 2) * 2 * C_::STAGE_TILE};
        typename Work::State state;
        int it = 0;
        while (more)
        {
            if (!t.skip)
            {
                Work::before(p, t, state, row0, col0, st, lane, abort);
            }
            const bool more_next = Work::tile(p, cid, clusters, ++i, next);
            for (int k0 = 0; !t.skip && k0 < t.kbs; k0 += SPLIT ? Work::CHAIN : t.kbs)
            {
                const int buf = TWO ? it & 1 : 0;
                warp_wait(&tfull[buf], (TWO ? it >> 1 : it) & 1, p.status, abort);
                fence_after();
                const uint32_t base = tmem + static_cast<uint32_t>(buf * TN + col0) +
                                      (static_cast<uint32_t>(quarter * 32) << 16);
                const bool last = !SPLIT || k0 + Work::CHAIN >= t.kbs;
                if constexpr (SPLIT)
                {
                    if (t.kbs > Work::CHAIN)
                    {
                        fold<COLS>(base, base - buf * TN + (TWO ? 2 : 1) * TN, k0 == 0, last);
                    }
                }
                if (last)
                {
                    Work::template epilogue<COLS>(p, t, state, base, row0, col0, st, lane);
                }
                fence_before();
                __syncwarp();
                if (lane == 0)
                {
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                     release + static_cast<uint32_t>(buf * 8))
                                 : "memory");
                }
                if (last)
                {
                    Work::after(p, t, lane);
                }
                ++it;
            }
            t = next;
            more = more_next;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");   // copies an epilogue left in flight
        if (lane == 0)
        {
            bulk_wait_group<0>();   // staged output fully written before the CTA's memory goes
        }
    }
    fence_before();
    __syncthreads();
    if (*abort != 0)
    {
        // a wait gave up: half a millisecond, in which the loads and products in flight end
        for (const long long start = clock64(); clock64() - start < (1ll << 20);)
        {
        }
    }
    cluster_sync();   // no CTA leaves while its peer may still read its operands or barriers
    __syncwarp();
    if (warp == 1)
    {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ---- host ------------------------------------------------------------------------------------
// A tensor map over `planes` row-major matrices of `rows` x `cols` (element size es: 2 for 16-bit,
// 4 for fp32), rows ld elements and planes `plane` elements apart, with boxes of bx x by (bx of at
// most the swizzle's bytes). The base must be 16-byte aligned, ld and plane multiples of 16 bytes.
enum class Swizzle { kNone, k64, k128 };
bool make_map3(CUtensorMap* map, const void* base, int es, bool is_bf16, int64_t cols, int64_t rows,
               int64_t planes, int64_t ld, int64_t plane, uint32_t bx, uint32_t by,
               Swizzle swizzle = Swizzle::k128);

// Shared memory of a launch: all of an SM's, so that no other kernel's blocks run beside it.
constexpr int kOwnSm = 227 * 1024;

// Clusters of the kernel that the current device can hold at once, capped by the SMs that
// veda_set_reserved_sms leaves (0: none fit; -1: the query failed, and is asked again at the next call).
// Cached per device.
template <class Work, int EPI_WARPS, bool SPLIT>
int clusters_available()
{
    constexpr int kDevices = 64;
    static std::atomic<int> cached[kDevices];   // 0: not asked yet, else clusters + 1
    int device = 0;
    cudaGetDevice(&device);
    if (device < 0 || device >= kDevices)
    {
        return 0;
    }
    int have = cached[device].load(std::memory_order_acquire);
    if (have == 0)
    {
        auto kernel = pair_kernel<Work, EPI_WARPS, SPLIT>;
        int n = 0;
        bool ok = false;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kOwnSm) == cudaSuccess)
        {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(2 * (sm_count() / 2));
            cfg.blockDim = dim3(Cfg<EPI_WARPS, Work::TN>::THREADS);
            cfg.dynamicSmemBytes = kOwnSm;
            cudaLaunchAttribute attr{};
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 2;
            attr.val.clusterDim.y = 1;
            attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            ok = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess;
        }
        if (!ok)
        {
            cudaGetLastError();
            return -1;
        }
        have = n + 1;
        cached[device].store(have, std::memory_order_release);
    }
    const int cap = compute_sms() / 2;
    return have - 1 < cap ? have - 1 : cap;
}

// The error of a call whose clusters_available() is below 1.
inline int none_available(const char* what, int clusters)
{
    return clusters < 0 ? fail(VEDA_ERR_CUDA, std::string(what) + ": the query for the device's clusters failed")
                        : fail(VEDA_ERR_UNSUPPORTED, std::string(what) + ": no CTA pair fits on this device");
}

// overlapped: may start while the kernel ahead is running (launch()), which has to be of this kind too: its blocks own
// their SMs as these do. Behind others the tensor memory would be allocated beside their last blocks, and there one
// cluster's allocation never came back, its SMs long empty and every other cluster finished: once in some 7000 calls
// of the loss head of 2048 x 32000 x 1024 in fp32, behind the launch that lays operands out. With both kept apart,
// 109000 calls ran through.
template <class Work, int EPI_WARPS, bool SPLIT>
int launch_pair(const char* what, const typename Work::Params& p, int clusters, bool overlapped, cudaStream_t s)
{
    const auto kernel = pair_kernel<Work, EPI_WARPS, SPLIT>;
    const dim3 grid(2 * clusters), block(Cfg<EPI_WARPS, Work::TN>::THREADS);
    if (overlapped)
    {
        return launch(what, kernel, grid, block, kOwnSm, s, p);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = kOwnSm;
    cfg.stream = s;
    count_launch();
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
    if (err != cudaSuccess)
    {
        cudaGetLastError();
        return fail(VEDA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(err));
    }
    return check_launch(what);
}

// The same with all clusters on the device at once (a cooperative launch), for a Work whose tiles wait
// for one another. Such a launch does not start before its predecessor has ended.
template <class Work, int EPI_WARPS, bool SPLIT>
int launch_together(const char* what, const typename Work::Params& p, int clusters, cudaStream_t s)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * clusters);
    cfg.blockDim = dim3(Cfg<EPI_WARPS, Work::TN>::THREADS);
    cfg.dynamicSmemBytes = kOwnSm;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeCooperative;
    attr.val.cooperative = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    count_launch();
    const cudaError_t err = cudaLaunchKernelEx(&cfg, pair_kernel<Work, EPI_WARPS, SPLIT>, p);
    if (err != cudaSuccess)
    {
        cudaGetLastError();
        return fail(VEDA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(err));
    }
    return check_launch(what);
}

} // namespace veda::cuda::pair
