// tcgen05 GEMM of the operators: C[M,N] = A[M,K] . B[N,K]^T in bf16 or f16 with fp32 accumulation
// in tensor memory, fed by TMA, by single CTAs or by pairs of CTAs on two SMs (CG = 1, 2).
//
// A pair works on one 256 x BN tile: each CTA holds 128 rows of A, half of the tile's B rows and a
// 128 x BN accumulator in its own tensor memory, and the first CTA's MMA warp issues
// tcgen05.mma.cta_group::2 for both. Each SM so stages 16 KB of A and BN * 64 B of B for a 64-wide
// k-block where a single CTA's 128 x BN tile needs BN * 128 B of B: at BN = 256, 32 KB for 512
// cycles of MMA against 48 KB.
//
// Warps of a CTA (576 threads, persistent over work items = tile x k split):
//   warp 0     TMA producer: waits for its own empty[stage], loads its CTA's A and B parts; the
//              bytes of both CTAs are counted by the first CTA's full[stage];
//   warp 1     (first CTA) MMA issuer: commits each stage to empty[stage] of both CTAs, a finished
//              accumulator to acc_full[buffer] of both;
//   warps 2-17 epilogue, in two sets of eight: a set takes every second tile, the one whose
//              accumulator is its buffer. quarter = warp % 4 gives the 32 tensor-memory lanes (rows),
//              group half of the columns; each warp arrives once at the first CTA's acc_empty.
// Two accumulator buffers of BN columns let the epilogue of one tile overlap the MMAs of the next. An
// epilogue is a chain of latencies (tensor memory, special functions, staging, its stores), so two
// tiles' chains run side by side, and not sixteen warps on one: 75,776 x 512 to 2,816 columns took
// 199 us with all warps on a tile and takes 188 (1,164 TFLOP/s; the library's product 187); without
// any epilogue 147. At 2,048 in k it is 594 us (1,471 TFLOP/s, library 592), with the SMs' clock held
// near 1.4 GHz by the power limit.
// Operands are K-major (rows of K elements) or MN-major (K rows), see gemm.cuh.
//
// Every wait is bounded: a stall is counted; the first CTA then waits (bounded) for the
// loads in flight, the CTAs meet, free their tensor memory and return.
#pragma once

#include <cuda.h>

#include "gemm.cuh"
#include "ops.cuh"

namespace t8b {
namespace op {

constexpr int kEpiWarps = 16, kSetWarps = 8;
constexpr int kGemmThreads = 64 + 32 * kEpiWarps;
constexpr int kStaging = 4096;  // an epilogue warp's staging: 32 rows of 128 bytes

// ------------------------------------------------------------------ PTX of the pair form
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The first CTA's copy of a barrier, as a shared::cluster address.
__device__ __forceinline__ uint32_t first_cta_addr(const void* p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tc::smem_addr(p)));
    return r;
}
__device__ __forceinline__ void cluster_arrive_wait() {
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
template <int CG>
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    if (CG == 1) {
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                         tc::smem_addr(dst)),
                     "l"(map), "r"(bar), "r"(x), "r"(y)
                     : "memory");
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                tc::smem_addr(dst)),
            "l"(map), "r"(bar), "r"(x), "r"(y)
            : "memory");
    }
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (CG == 1) {
        tc::mma(d, a, b, idesc, accumulate);
    } else {
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    }
}
// Signals the barrier at this offset in every CTA of the group once the MMAs so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if (CG == 1) {
        tc::commit(bar);
    } else {
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                tc::smem_addr(bar)),
            "h"(static_cast<uint16_t>(3))
            : "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {
    if (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_addr(slot)), "r"(columns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_addr(slot)), "r"(columns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    if (CG == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
    } else {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
    }
}

// kind::f16 instruction descriptor: fp32 accumulators, A and B both bf16 or both f16.
template <typename E>
__host__ __device__ constexpr uint32_t instruction(int m, int n, bool a_mn, bool b_mn) {
    const uint32_t format = Element<E>::kType == T8B_BF16 ? 1u : 0u;
    return (1u << 4) | (format << 7) | (format << 10) | (static_cast<uint32_t>(a_mn) << 15) |
        (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// ------------------------------------------------------------------ epilogue staging
// A staging tile holds 32 rows of BYTES (64 or 128) bytes in 16-byte pieces, laid out as the TMA
// swizzle of that width lays them out, so one box moves it and lanes that each touch a piece of
// their own row meet no bank twice.
template <int BYTES>
__device__ __forceinline__ unsigned char* piece(unsigned char* tile, int row, int q) {
    return BYTES == 128 ? tile + row * 128 + ((q ^ (row & 7)) << 4) : tile + row * 64 + ((q ^ ((row >> 1) & 3)) << 4);
}

// A matrix that epilogues read or write, 32 rows at a time. `tma`: rows start on 16-byte
// boundaries, and map moves tiles of 32 rows by BYTES bytes; otherwise element by element.
struct Tiled {
    CUtensorMap map;
    void* data;
    int64_t stride;
    int rows, columns;
    int tma;
};

// Sends a staging tile (rows row0.., columns col0.. of m), written by all lanes, out: by TMA, or
// element by element. The tile may be written again after free_tile().
template <typename T, int BYTES>
__device__ __forceinline__ void send(const Tiled& m, unsigned char* tile, int row0, int col0, int lane) {
    if (m.tma) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            if (row0 < m.rows && col0 < m.columns) tc::tma_store(&m.map, tile, col0, row0);
            tc::bulk_commit();
        }
        return;
    }
    __syncwarp();
    constexpr int W = BYTES / sizeof(T);
    constexpr int kPer = 16 / sizeof(T);
    const int rows = min(32, m.rows - row0);
    T* out = static_cast<T*>(m.data) + static_cast<int64_t>(row0) * m.stride + col0;
    for (int r = 0; r < rows; ++r, out += m.stride) {
#pragma unroll
        for (int c = lane; c < W; c += 32) {
            if (col0 + c < m.columns) out[c] = reinterpret_cast<const T*>(piece<BYTES>(tile, r, c / kPer))[c % kPer];
        }
    }
    __syncwarp();
}
// This warp's stores have read its staging tile.
__device__ __forceinline__ void free_tile(int lane) {
    if (lane == 0) tc::bulk_wait_read();
    __syncwarp();
}

// Fetches a tile of m into a free staging tile; by TMA it arrives on `bar` (lane 0 waits).
template <typename T, int BYTES>
__device__ __forceinline__ void fetch(const Tiled& m, unsigned char* tile, uint64_t* bar, int row0, int col0, int lane) {
    if (m.tma) {
        if (lane == 0) {
            tc::bar_expect(bar, 32 * BYTES);
            tc::tma_load(tile, &m.map, bar, col0, row0);
        }
        return;
    }
    constexpr int W = BYTES / sizeof(T);
    constexpr int kPer = 16 / sizeof(T);
    const int rows = min(32, m.rows - row0);
    const T* in = static_cast<const T*>(m.data) + static_cast<int64_t>(row0) * m.stride + col0;
    for (int r = 0; r < rows; ++r, in += m.stride) {
#pragma unroll
        for (int c = lane; c < W; c += 32) {
            if (col0 + c < m.columns) reinterpret_cast<T*>(piece<BYTES>(tile, r, c / kPer))[c % kPer] = in[c];
        }
    }
    __syncwarp();
}

// What an epilogue sees: one warp of a tile.
struct Warp {
    int row0;             // first of the warp's 32 rows
    int tn;               // the tile's index along the columns
    int split, group, lane;
    uint32_t taddr;       // the warp's lanes of the tile's accumulator
    unsigned char* tile;  // its staging, kStaging bytes
    float* vector;        // 32 floats for a bias
    uint64_t* bar;        // a fetch's arrival
    uint32_t phase;       // its parity
    bool in_flight;       // a fetch not waited for yet
    volatile int* abort;

    // the fetch has arrived
    __device__ __forceinline__ bool wait() {
        const bool ok = tc::bar_wait(bar, phase, abort);
        phase ^= 1u;
        in_flight = false;
        return ok;
    }
};

// An epilogue's wait for its accumulator: it sleeps between polls, which leaves the issue slots and
// some of the chip's power to the tile in progress (75,776 x 1,024 to 512 columns: 70 -> 67 us).
__device__ __forceinline__ bool wait_idle(uint64_t* bar, uint32_t parity, volatile int* abort) {
    for (uint32_t i = 0; i < tc::kSpinLimit; ++i) {
        if (tc::bar_try(bar, parity)) return true;
        if (*abort) return false;
        __nanosleep(100);
    }
    return false;
}

// Polls a CTA that gives up makes for the loads it has in flight.
constexpr uint32_t kDrainLimit = 1u << 18;

struct Shape {
    int tiles_m, tiles_n, splits, k_blocks;
    int second;  // B's second half starts at this row (gated projections); 0: B is one matrix
    int after;   // what the kernel before this one is to it: kInput or kBeside
    unsigned* stalls;  // the device's count of waits that ran out
};

// A CTA's (or pair's) work items, one in `step`, columns fastest, then rows, then parts of k. Each
// item is the last one plus a fixed step in the mixed radix, so the one thread that issues the MMAs
// does not divide between tiles.
struct Walk {
    int tiles_m, tiles_n, splits, k_blocks;
    int dn, dm, ds;
    int tn, tm, split, kb0, kb1;
    __device__ __forceinline__ Walk(const Shape& s, int first, int step)
        : tiles_m(s.tiles_m), tiles_n(s.tiles_n), splits(s.splits), k_blocks(s.k_blocks) {
        dn = step % tiles_n;
        dm = step / tiles_n % tiles_m;
        ds = step / tiles_n / tiles_m;
        tn = first % tiles_n;
        tm = first / tiles_n % tiles_m;
        split = first / tiles_n / tiles_m;
        range();
    }
    __device__ __forceinline__ bool more() const { return split < splits; }
    __device__ __forceinline__ void next() {
        const int before = split;
        tn += dn;
        if (tn >= tiles_n) {
            tn -= tiles_n;
            ++tm;
        }
        tm += dm;
        if (tm >= tiles_m) {
            tm -= tiles_m;
            ++split;
        }
        split += ds;
        if (split != before) range();
    }
    __device__ __forceinline__ void range() {  // k_blocks * (splits + 1) fits 32 bits
        kb0 = splits == 1 ? 0 : static_cast<int>(static_cast<uint32_t>(k_blocks) * split / splits);
        kb1 = splits == 1 ? k_blocks : static_cast<int>(static_cast<uint32_t>(k_blocks) * (split + 1) / splits);
    }
};

template <int CG, int BN>
struct Plan {
    static constexpr int kABytes = tc::BM * tc::BK * 2;
    static constexpr int kBRows = BN / CG;
    static constexpr int kBBytes = kBRows * tc::BK * 2;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kEpiBytes = kEpiWarps * (kStaging + 128);
    static constexpr int kBarBytes = 384;
    static constexpr int kBudget = 232448 - kEpiBytes - kBarBytes;
    static constexpr int kStages = kBudget / kStageBytes > 8 ? 8 : kBudget / kStageBytes;
    static constexpr int kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
    static constexpr int kSmemBytes = kStages * kStageBytes + kEpiBytes + kBarBytes;
    static_assert(kStages >= 3, "at least three stages");
    static_assert(kBarBytes >= (2 * kStages + 4 + kEpiWarps) * 8 + 8, "barriers");
};

template <typename E, int CG, int BN, bool A_MN, bool B_MN, class Epi>
__global__ void __cluster_dims__(CG, 1, 1) __launch_bounds__(kGemmThreads, 1)
    k_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Shape s,
           const __grid_constant__ Epi epi) {
    using P = Plan<CG, BN>;
    extern __shared__ __align__(1024) unsigned char base[];
    unsigned char* epi_tiles = base + P::kStages * P::kStageBytes;
    float* vectors = reinterpret_cast<float*>(epi_tiles + kEpiWarps * kStaging);
    uint64_t* full = reinterpret_cast<uint64_t*>(epi_tiles + P::kEpiBytes);
    uint64_t* empty = full + P::kStages;
    uint64_t* acc_full = empty + P::kStages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* fetched = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fetched + kEpiWarps);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    if ((tc::smem_addr(base) & 1023u) != 0) {  // the swizzles count on it; every thread sees the same
        if (threadIdx.x == 0) atomicAdd(s.stalls, 1u);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 1 ? 0 : static_cast<int>(cluster_rank());
    if (threadIdx.x == 0) {
        for (int i = 0; i < P::kStages; ++i) {
            tc::bar_init(full + i, 1);
            tc::bar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::bar_init(acc_full + i, 1);
            tc::bar_init(acc_empty + i, CG * kSetWarps);
        }
        for (int i = 0; i < kEpiWarps; ++i) tc::bar_init(fetched + i, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_alloc<CG>(tmem_slot, P::kTmemCols);
    tc::fence_before();
    __syncthreads();
    if (CG == 2) cluster_arrive_wait();  // the peer's barriers are initialised
    tc::fence_after();
    if (s.after == kInput) wait_previous();
    release_next();
    const uint32_t tmem = *tmem_slot;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    auto stop = [&]() {
        *abort = 1;
        atomicAdd(s.stalls, 1u);
    };

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, started = 0;
            uint32_t phase = 0;
            for (Walk t(s, first, step); t.more() && !*abort; t.next()) {
                const int row = (t.tm * CG + rank) * tc::BM;
                for (int kb = t.kb0; kb < t.kb1; ++kb) {
                    if (!tc::bar_wait(empty + stage, phase ^ 1u, abort)) {
                        stop();
                        break;
                    }
                    unsigned char* a = base + stage * P::kStageBytes;
                    unsigned char* b = a + P::kABytes;
                    const uint32_t bar = CG == 1 ? tc::smem_addr(full + stage) : first_cta_addr(full + stage);
                    if (rank == 0) tc::bar_expect(full + stage, CG * P::kStageBytes);
                    if (A_MN) {
#pragma unroll
                        for (int j = 0; j < tc::BM / 64; ++j) load_tile<CG>(a + j * 8192, &map_a, bar, row + j * 64, kb * tc::BK);
                    } else {
                        load_tile<CG>(a, &map_a, bar, kb * tc::BK, row);
                    }
                    if (B_MN) {
#pragma unroll
                        for (int j = 0; j < P::kBRows / 64; ++j) {
                            load_tile<CG>(b + j * 8192, &map_b, bar, t.tn * BN + rank * P::kBRows + j * 64, kb * tc::BK);
                        }
                    } else if (s.second == 0) {
                        load_tile<CG>(b, &map_b, bar, kb * tc::BK, t.tn * BN + rank * P::kBRows);
                    } else if (CG == 2) {
                        load_tile<CG>(b, &map_b, bar, kb * tc::BK, rank * s.second + t.tn * (BN / 2));
                    } else {
                        load_tile<CG>(b, &map_b, bar, kb * tc::BK, t.tn * (BN / 2));
                        load_tile<CG>(b + P::kBBytes / 2, &map_b, bar, kb * tc::BK, s.second + t.tn * (BN / 2));
                    }
                    if (started < P::kStages) ++started;
                    if (++stage == P::kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (*abort && rank == 0) {  // the loads in flight land before the CTA ends (each wait bounded)
                for (int i = 0; i < started; ++i) {
                    if (--stage < 0) {
                        stage = P::kStages - 1;
                        phase ^= 1u;
                    }
                    for (uint32_t n = 0; n < kDrainLimit && !tc::bar_try(full + stage, phase); ++n) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && lane == 0) {
            constexpr uint32_t idesc = instruction<E>(tc::BM * CG, BN, A_MN, B_MN);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            for (Walk t(s, first, step); t.more() && !*abort; t.next()) {
                if (!tc::bar_wait(acc_empty + acc, acc_phase ^ 1u, abort)) {
                    stop();
                    break;
                }
                tc::fence_after();
                const uint32_t d = tmem + static_cast<uint32_t>(acc * BN);
                bool ok = true;
                for (int kb = t.kb0; kb < t.kb1; ++kb) {
                    if (!tc::bar_wait(full + stage, phase, abort)) {
                        stop();
                        ok = false;
                        break;
                    }
                    tc::fence_after();
                    const uint32_t a = tc::smem_addr(base + stage * P::kStageBytes);
                    const uint32_t b = a + P::kABytes;
#pragma unroll
                    for (int k = 0; k < tc::BK / 16; ++k) {
                        const uint64_t da = A_MN ? tc::sw128_desc(a + k * 2048, 8192, 1024) : tc::sw128_desc(a + k * 32, 16, 1024);
                        const uint64_t db = B_MN ? tc::sw128_desc(b + k * 2048, 8192, 1024) : tc::sw128_desc(b + k * 32, 16, 1024);
                        mma<CG>(d, da, db, idesc, (kb > t.kb0 || k > 0) ? 1u : 0u);
                    }
                    commit<CG>(empty + stage);
                    if (++stage == P::kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                commit<CG>(acc_full + acc);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
    } else {
        const int e = warp - 2, quarter = warp & 3, acc = e / kSetWarps;
        Warp w;
        w.group = (e >> 2) & 1;
        w.lane = lane;
        w.tile = epi_tiles + e * kStaging;
        w.vector = vectors + e * 32;
        w.bar = fetched + e;
        w.phase = 0;
        w.in_flight = false;
        w.abort = abort;
        w.taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BN);
        uint32_t acc_phase = 0;
        Walk t(s, first, step);
        if (acc == 1) t.next();
        for (; t.more() && !*abort; t.next(), t.next(), acc_phase ^= 1u) {
            w.row0 = (t.tm * CG + rank) * tc::BM + quarter * 32;
            w.tn = t.tn;
            w.split = t.split;
            epi.begin(w);
            if (!wait_idle(acc_full + acc, acc_phase, abort)) {
                stop();
                break;
            }
            tc::fence_after();
            if (!epi.finish(w)) {
                stop();
                break;
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 1) {
                    tc::bar_arrive(acc_empty + acc);
                } else {
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(first_cta_addr(acc_empty + acc))
                                 : "memory");
                }
            }
        }
        for (uint32_t n = 0; w.in_flight && n < kDrainLimit && !tc::bar_try(w.bar, w.phase); ++n) {  // after a stall
        }
        if (lane == 0) tc::bulk_wait();  // this warp's stores have landed
        __syncwarp();
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (CG == 2) cluster_arrive_wait();  // no CTA of a pair ends while the other may still signal it
    if (s.after == kBeside) wait_previous();  // the next kernel's wait for this one covers both
    if (warp == 2) {
        tc::fence_after();
        tmem_free<CG>(tmem, P::kTmemCols);
    }
}

}  // namespace op
}  // namespace t8b
