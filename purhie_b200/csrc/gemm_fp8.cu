// The matrix product of 8-bit operands with scales, on the 5th-generation tensor cores:
//
//   out[m, n] = sum_b xs[m, b] * ws[n / 128, b] * sum_{k in block b} x[m, k] * w[n, k],
//
// x [M, K] rows in e4m3 with a float32 scale for each 128 values, w [N, K] a weight in e4m3 with a scale for each block of
// 128 x 128, both K-major.  The inner sum, over the 128 values that share their scales, is four tcgen05.mma (kind::f8f6f4, 32
// of K each) into an accumulator in tensor memory that starts from zero; the outer one is float32, in registers: the epilogue
// warps read each block's accumulator with tcgen05.ld, multiply it by the two scales and add, while the tensor cores work on
// the next blocks in other accumulators.  A block of K is one stage of the ring: 128 bytes a row, one row of the swizzle.
//
// One CTA computes 128 features x BN tokens: the weight, which is what has to be streamed when tokens are few, fills the 128
// rows of the instruction, a thread's scale differs by column and comes from shared memory, and the lanes of a warp hold
// neighbouring features, so that whole lines leave straight from the registers.  Where the tiles are fewer than the CTAs that the
// device holds, K is cut into parts: float32 sums [part][token][feature] that whoever consumes the product adds up in order
// (the norm and the activation take them), or a short kernel behind this one; the same bits every time.  (Cut among the CTAs of
// a cluster that add up in shared memory, 8 x 6144 x 4096 took 16 us: a cluster starts late and not under the kernel in front.
// With mma.sync and 16 features a CTA, K whole, 8 x 24576 x 4096 took 25 us: its 8-bit products are slow here.)
// Many tokens: pairs of CTAs, further down; theirs can end in a gated activation.
//
// Every wait on an mbarrier is bounded; a wait that runs out sets *error_flag, and the CTA still frees its tensor memory and
// returns (what it writes is then meaningless).
// The reference's counterpart is its WMMA tile kernel over 8-bit blocks (src/matvec_q.hip:3437-3547).
#include "common.cuh"
#include "fp8_values.cuh"
#include "mbarrier.cuh"
#include "shared_limit.cuh"

#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <mutex>

namespace {

using namespace ph;
using ph_mbar::arrive;
using ph_mbar::arrive_expect_tx;
using ph_mbar::fence_init;
using ph_mbar::init;
using ph_mbar::smem_addr;

constexpr int BM = 128;
constexpr int BK = 128;                     // values (bytes) of K in a stage: one block of the scales
constexpr int UMMA_K = 32;
constexpr int THREADS = 192;                // copies, products, four epilogue warps
constexpr int A_BYTES = BM * BK;
constexpr int FACTOR_BLOCKS = 32;           // blocks of K whose factors lie in shared memory at a time
constexpr int MAX_SPLITS = 16;
constexpr int MAX_SIZE = 1 << 30;           // of M, N and K: tiles and blocks are counted in 32 bits

#define PH_ERR_FP8_PRODUCER 131
#define PH_ERR_FP8_MMA 132
#define PH_ERR_FP8_EPILOGUE 133

struct Params {
    const float* xs;
    const float* ws;
    void* out;
    int out_bf16;
    int M, N;
    int kblocks;
    int a_tiles, splits;
    int early_w;
    // Pairs, the gated activation in the epilogue: w's rows are (gate, up) pairs, out is [M, N / 2] in e4m3 with out_scales [M, N / 256]
    float* out_scales;
    ph_fp8::Gate gate;
    int tma_store;               // pairs: the copy engine stores; 0: the threads do
    int* error_flag;
};

// Where a wait that ran out is noted when the caller has no place of its own for it (one for each device).
__device__ int g_error;
__device__ __forceinline__ int* error_word(const Params& p) { return p.error_flag ? p.error_flag : &g_error; }

// A bounded wait that looks at the clock only now and then: these waits are short and follow one another, and the clock is slow to
// read.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* flag, int code) {
    unsigned long long t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (ph_mbar::try_wait(bar, parity)) return true;
        if ((i & 255u) == 0) {
            const unsigned long long now = ph_mbar::global_timer();
            if (t0 == 0) t0 = now;
            else if (now - t0 > ph_mbar::WAIT_LIMIT_NS) {
                atomicExch(flag, code);
                return false;
            }
        }
    }
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c_inner, int c_row) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(smem_addr(bar)), "r"(c_inner), "r"(c_row) : "memory");
}
// A tile's way from memory to L2 alone.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int c_inner, int c_row) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c_inner), "r"(c_row) : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void umma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}

// Shared-memory matrix descriptor of a K-major tile with the 128-byte swizzle: address >> 4 in bits 0-13, groups of eight rows 1024
// bytes apart (>> 4, bits 32-45), version 1 at bit 46, swizzle mode 2 at bits 61-63.
__device__ __forceinline__ uint64_t smem_desc(const void* p) {
    return (uint64_t)((smem_addr(p) & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor, kind::f8f6f4: D float32 (bits 4-5 = 1), A and B e4m3 (bits 7-9, 10-12 = 0), both K-major, N >> 3 at
// bits 17-22, M >> 4 at bits 24-28.
__host__ __device__ constexpr uint32_t make_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Two CTAs share an SM, so that one's start and end overlap the other's streaming.
template <int BN> struct Tile {
    static constexpr int STAGE_BYTES = A_BYTES + BN * BK;
    static constexpr int CTAS_PER_SM = 2;
    static constexpr int STAGES = 96 * 1024 / STAGE_BYTES;
    static constexpr int TMEM_COLS = BN >= 64 ? 256 : 128;
    static constexpr int BUFFERS = TMEM_COLS / BN;                       // accumulators in tensor memory
    static constexpr int FACTORS_LD = BN + 4;                            // (lanes write down a column: on eight banks, not on one)
    static constexpr int FACTORS_BYTES = FACTOR_BLOCKS * FACTORS_LD * 4;
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + FACTORS_BYTES + 256;
    static constexpr int CHUNK = BN >= 64 ? 32 : 16;                     // columns of an accumulator that are read at a time
    static_assert(TMEM_COLS * CTAS_PER_SM <= 512, "tensor memory");
    static_assert((2 * STAGES + 2 * BUFFERS) * 8 + 4 <= 256, "barriers");
};

template <int BN>
__global__ void __launch_bounds__(THREADS, Tile<BN>::CTAS_PER_SM)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, Params p) {
    using Cfg = Tile<BN>;
    constexpr int STAGES = Cfg::STAGES, BUFFERS = Cfg::BUFFERS, CHUNK = Cfg::CHUNK;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* smem_w = smem;
    uint8_t* smem_x = smem + STAGES * A_BYTES;
    float* factors = (float*)(smem + STAGES * Cfg::STAGE_BYTES);         // [block][token]
    uint64_t* full = (uint64_t*)(smem + STAGES * Cfg::STAGE_BYTES + Cfg::FACTORS_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + BUFFERS;
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + BUFFERS);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { init(&full[s], 1); init(&empty[s], 1); }
        for (int b = 0; b < BUFFERS; ++b) { init(&acc_full[b], 1); init(&acc_empty[b], 4); }
        fence_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    int* flag = error_word(p);
    const int splits = p.splits, split = blockIdx.x % splits, tile = blockIdx.x / splits;
    const int n0 = (tile % p.a_tiles) * BM, m0 = (tile / p.a_tiles) * BN;
    const int kb0 = (int)((long long)p.kblocks * split / splits), kb1 = (int)((long long)p.kblocks * (split + 1) / splits);

    pdl_launch_dependents();
    if (warp == 0) {
        if (lane == 0) {
            // the weight's tiles of the first stages may not have to wait for the kernel in front
            int pre = 0;
            if (p.early_w)
                for (; pre < STAGES && kb0 + pre < kb1; ++pre) {
                    arrive_expect_tx(&full[pre], Cfg::STAGE_BYTES);
                    tma_load_2d(smem_w + pre * A_BYTES, &map_w, &full[pre], (kb0 + pre) * BK, n0);
                }
            else if (splits > 1) {
                // A weight that may still be written can be on its way to L2 all the same: what is read there afterwards is what it
                // is by then.  (Where K is whole a CTA streams long enough: 8 x 24576 x 4096 18.6 us, 19.4 with this; in nine parts
                // 8 x 4096 x 12288 13.5 us, 12.2 with this.)
                for (int kb = kb0; kb < kb1 && kb < kb0 + 4; ++kb) tma_prefetch_2d(&map_w, kb * BK, n0);
            }
            pdl_wait();
            for (int s = 0; s < pre; ++s) tma_load_2d(smem_x + s * BN * BK, &map_x, &full[s], (kb0 + s) * BK, m0);
            int stage = pre == STAGES ? 0 : pre;
            uint32_t phase = pre == STAGES ? 1 : 0;
            bool ok = true;
            for (int kb = kb0 + pre; kb < kb1; ++kb) {
                if (!wait(&empty[stage], phase ^ 1, flag, PH_ERR_FP8_PRODUCER)) { ok = false; break; }
                arrive_expect_tx(&full[stage], Cfg::STAGE_BYTES);
                tma_load_2d(smem_w + stage * A_BYTES, &map_w, &full[stage], kb * BK, n0);
                tma_load_2d(smem_x + stage * BN * BK, &map_x, &full[stage], kb * BK, m0);
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
            // not past this point while copies may be in flight: the products have released every stage, or, after a wait that ran
            // out, the copies have at least arrived
            for (int s = 0; s < STAGES; ++s) {
                if (ok && !wait(&empty[stage], phase ^ 1, flag, PH_ERR_FP8_PRODUCER)) ok = false;
                if (!ok) wait(&full[stage], phase ^ 1, flag, PH_ERR_FP8_PRODUCER);
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = make_idesc(BM, BN);
            int stage = 0, buf = 0;
            uint32_t phase = 0, buf_phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait(&acc_empty[buf], buf_phase ^ 1, flag, PH_ERR_FP8_MMA) || !wait(&full[stage], phase, flag, PH_ERR_FP8_MMA)) break;
                tc_fence_after();
                const uint64_t adesc = smem_desc(smem_w + stage * A_BYTES), bdesc = smem_desc(smem_x + stage * BN * BK);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k)                    // 32 values further along the swizzled row
                    umma(tmem_base + (uint32_t)(buf * BN), adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), idesc, k > 0 ? 1u : 0u);
                umma_commit(&acc_full[buf]);
                umma_commit(&empty[stage]);
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
                if (++buf == BUFFERS) { buf = 0; buf_phase ^= 1; }
            }
        }
    } else {
        const int q = warp & 3;                                          // the quarter of the accumulator's rows that this warp may read
        const int n = n0 + q * 32 + lane;
        pdl_wait();
        float acc[BN];
#pragma unroll
        for (int j = 0; j < BN; ++j) acc[j] = 0.0f;
        int buf = 0;
        uint32_t buf_phase = 0;
        bool ok = true;
        const float* ws = p.ws + (size_t)(n0 / BK) * p.kblocks;
        for (int base = kb0; base < kb1; base += FACTOR_BLOCKS) {
            // the factors of the next blocks of K, [block][token], each the product of both scales: a lane a block, a warp a token
            const int some = min(FACTOR_BLOCKS, kb1 - base);
            if (base > kb0) asm volatile("bar.sync 1, 128;" ::: "memory");
            if (lane < some) {
                float v[BN / 4];
#pragma unroll
                for (int i = 0; i < BN / 4; ++i) v[i] = p.xs[(size_t)min(m0 + warp - 2 + 4 * i, p.M - 1) * p.kblocks + base + lane];
                const float s = ws[base + lane];
#pragma unroll
                for (int i = 0; i < BN / 4; ++i) factors[lane * Cfg::FACTORS_LD + warp - 2 + 4 * i] = v[i] * s;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int b = 0; b < some; ++b) {
                const float4* f = (const float4*)(factors + b * Cfg::FACTORS_LD);
                ok = ok && wait(&acc_full[buf], buf_phase, flag, PH_ERR_FP8_EPILOGUE);
                __syncwarp();
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN);
                uint32_t r[2][CHUNK];
                if constexpr (CHUNK == 32) tmem_ld32(taddr, r[0]); else tmem_ld16(taddr, r[0]);
#pragma unroll
                for (int c = 0; c < BN / CHUNK; ++c) {
                    tmem_ld_wait();
                    if (c + 1 < BN / CHUNK) {
                        if constexpr (CHUNK == 32) tmem_ld32(taddr + (c + 1) * CHUNK, r[(c + 1) & 1]); else tmem_ld16(taddr + (c + 1) * CHUNK, r[(c + 1) & 1]);
                    } else {
                        tc_fence_before();                               // all of it is in registers: the accumulator is free
                        __syncwarp();
                        if (lane == 0) arrive(&acc_empty[buf]);
                    }
#pragma unroll
                    for (int j = 0; j < CHUNK; j += 4) {
                        const float4 v = f[(c * CHUNK + j) / 4];
                        float* a = acc + c * CHUNK + j;
                        const uint32_t* d = r[c & 1] + j;
                        a[0] = fmaf(__uint_as_float(d[0]), v.x, a[0]); a[1] = fmaf(__uint_as_float(d[1]), v.y, a[1]);
                        a[2] = fmaf(__uint_as_float(d[2]), v.z, a[2]); a[3] = fmaf(__uint_as_float(d[3]), v.w, a[3]);
                    }
                }
                if (++buf == BUFFERS) { buf = 0; buf_phase ^= 1; }
            }
        }
        // the lanes of a warp hold neighbouring features of a token: whole lines leave straight from the registers
        if (p.out_bf16) {
            // (two tokens at a time: the even lanes store a pair of features of the one, the odd lanes of the other)
            const int odd = lane & 1, pair = n - odd;
            const bool wide = (p.N & 1) == 0 && ((uintptr_t)p.out & 3) == 0;
#pragma unroll
            for (int j = 0; j < BN; j += 2) {
                const float got = __shfl_xor_sync(0xffffffffu, odd ? acc[j] : acc[j + 1], 1);
                const __nv_bfloat162 v = odd ? __floats2bfloat162_rn(got, acc[j + 1]) : __floats2bfloat162_rn(acc[j], got);
                const int m = m0 + j + odd;
                if (m >= p.M || pair >= p.N) continue;
                __nv_bfloat16* o = (__nv_bfloat16*)p.out + (size_t)m * p.N + pair;
                if (wide) *(__nv_bfloat162*)o = v;
                else {
                    o[0] = __low2bfloat16(v);
                    if (pair + 1 < p.N) o[1] = __high2bfloat16(v);
                }
            }
        } else if (n < p.N) {
            float* o = (float*)p.out + (size_t)split * p.M * p.N + (size_t)m0 * p.N + n;
#pragma unroll
            for (int j = 0; j < BN; ++j)
                if (m0 + j < p.M) o[(size_t)j * p.N] = acc[j];
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    }
}

// out = the sum of the parts ([parts][values] float32), in their order; four values a thread.
template <typename T>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* __restrict__ parts, int n_parts, long long values, T* __restrict__ out) {
    pdl_launch_dependents();
    pdl_wait();
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= values) return;
    if ((values & 3) == 0 && ((uintptr_t)out & (4 * sizeof(T) - 1)) == 0) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int s = 0; s < n_parts; ++s) {
            const float4 a = *(const float4*)(parts + s * values + i);
            v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        }
        store4(out + i, v);
    } else {
        for (long long j = i; j < i + 4 && j < values; ++j) {
            float v = 0.0f;
            for (int s = 0; s < n_parts; ++s) v += parts[s * values + j];
            out[j] = from_float<T>(v);
        }
    }
}

// ---- two CTAs on one tile (cta_group::2) ---------------------------------------------------------------
//
// Many tokens: a cluster of two CTAs, on the two SMs of a pair, works on tiles of 256 tokens x 256 features, one pair per two
// SMs, tile after tile.  Each CTA copies its own 128 rows of x and 128 rows of w for a block of K, half of what a CTA alone
// would read from shared memory per product; the leader (rank 0) issues the products with M = 256, N = 256, which leave each
// CTA its own 128 tokens x 256 features in its tensor memory: two accumulators of 256 columns, all of it.  Eight epilogue warps, two for
// each quarter of the rows, keep the float32 sums of 32 tokens x 128 features a warp in registers, 128 a thread.
// What bounds it: the products alone, with the sums left in tensor memory, take 64 us for 2048 x 9472 x 4096 (2,470 TFLOP/s), with
// the accumulators read for each block 73, with the multiply-adds 79 (2,010): both sides are busy, and hand two accumulators back
// and forth.  Four accumulators of 128 columns were slower (92: a product of 128 columns reads its rows of x again).
//   full[s]      in the leader: the copies of both CTAs complete there, the leader's thread announces the bytes of both;
//   empty[s]     in each CTA: the leader's tcgen05.commit reaches both (the commit's own multicast; no load is multicast);
//   acc_full[a]  in each CTA, by the same kind of commit; acc_empty[a] in the leader, counted in by the epilogue warps of both.
constexpr int PAIR_BN = 256;
constexpr int PAIR_HALF = PAIR_BN / 2;
constexpr int PAIR_STAGE_BYTES = A_BYTES + PAIR_HALF * BK;
constexpr int PAIR_STAGES = 4;
constexpr int PAIR_WARPS = 8;
constexpr int PAIR_THREADS = 128 + 32 * PAIR_WARPS;
// Registers a thread: the launch gives each of the 384 threads 168 (what 65,536 hold), the four warps of copies and products hand
// most of theirs back and the epilogue's take them: 128 * 56 + 256 * 224 = 384 * 168.
constexpr int PAIR_REGS = 168, PAIR_REGS_LOW = 56, PAIR_REGS_HIGH = 224;
static_assert(128 * PAIR_REGS_LOW + 32 * PAIR_WARPS * PAIR_REGS_HIGH <= PAIR_THREADS * PAIR_REGS, "more registers than the launch has");
constexpr int PAIR_BOX_BYTES = 32 * 128;                          // 32 rows of 128 bytes on their way out
constexpr int PAIR_STAGING_BYTES = PAIR_WARPS * 2 * PAIR_BOX_BYTES;
constexpr int PAIR_GROUPS = 3;                                    // of four blocks of K, whose factors lie in shared memory
constexpr int PAIR_FACTORS_BYTES = PAIR_GROUPS * 2 * 4 * BM * 4;
constexpr int PAIR_SMEM_BYTES = 1024 + PAIR_STAGES * PAIR_STAGE_BYTES + PAIR_STAGING_BYTES + PAIR_FACTORS_BYTES + 256;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
    uint32_t out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_addr(p)), "r"(rank));
    return out;
}
// Relaxed: what it tells is that tensor memory has been read, which the tcgen05 fence in front orders; nothing in other memory is
// handed on.  With release semantics at cluster scope a warp waits for all it has in flight, most of a microsecond for each block of
// K: 2048 x 24576 x 4096 took 408 us.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c_inner, int c_row) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(bar), "r"(c_inner), "r"(c_row) : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier at this place in both CTAs when the products issued so far are complete.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_addr(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c_inner, int c_row, int c_part) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_addr(src)), "r"(c_inner), "r"(c_row), "r"(c_part)
                 : "memory");
}
// a += v * f on two values at once.
__device__ __forceinline__ void fma2(float& a0, float& a1, uint32_t v0, uint32_t v1, float f) {
    asm("{\n.reg .b64 a, v, f;\nmov.b64 a, {%0, %1};\nmov.b64 v, {%2, %3};\nmov.b64 f, {%4, %4};\nfma.rn.f32x2 a, v, f, a;\nmov.b64 {%0, %1}, a;\n}"
        : "+f"(a0), "+f"(a1) : "r"(v0), "r"(v1), "f"(f));
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
}

// A thread's 128 columns of its row as 64 gated values in 8 bits.  largest [turn][half][row of the CTA]: two turns, so that a warp that
// is a tile ahead does not write what its partner has yet to read.  Tiles are whole (N a multiple of 256).
__device__ __forceinline__ void store_gated(const Params& p, float* acc, float* largest, int turn, int q, int half, int lane, int row, int n0) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < PAIR_HALF / 2; ++j) {
        acc[j] = ph_fp8::gated_value(p.gate, acc[2 * j], acc[2 * j + 1]);
        m = ph_fp8::max_nan(m, fabsf(acc[j]));
    }
    float* at = largest + turn * 2 * BM + q * 32 + lane;
    at[half * BM] = m;
    asm volatile("bar.sync %0, 64;" ::"r"(2 + q) : "memory");
    const float a = ph_fp8::max_nan(ph_fp8::max_nan(m, at[(half ^ 1) * BM]), ph_fp8::LEAST);
    if (row >= p.M) return;
    const int F = p.N / 2;
    if (half == 0) p.out_scales[(size_t)row * (F / ph_fp8::BLOCK) + n0 / PAIR_BN] = a / ph_fp8::TOP;
    const float inverse = ph_fp8::TOP / a;
    uint4* o = (uint4*)((uint8_t*)p.out + (size_t)row * F + n0 / 2);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* h = acc + c * 16 + i * 4;
            v[i] = ph_fp8::pack2(h[0] * inverse, h[1] * inverse) | ph_fp8::pack2(h[2] * inverse, h[3] * inverse) << 16;
        }
        o[c] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

// GATED: the epilogue applies the gated activation and brings its values to 8 bits.  A tile's 256 features are 128 (gate, up) pairs, one
// block of the result for each of its rows: the two warps that hold a row's halves tell each other their largest magnitudes.  The tensor
// cores stand still while a tile's 64 exponentials a thread are made, but the product's 100 MB neither leave nor come back: in a graph, over
// weights that L2 does not hold, 512 x 24576 x 4096 takes 73 us and 75 as two kernels, 2,048 rows 252 and 258, 8,192 rows 915 and 942; a
// prompt of 2,048 tokens through 36 such layers, at the power limit, 22.7 ms for 23.25.
template <bool GATED>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out, Params p) {
    constexpr int STAGES = PAIR_STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* smem_a = smem;
    uint8_t* smem_b = smem + STAGES * A_BYTES;
    uint8_t* staging = smem + STAGES * PAIR_STAGE_BYTES;
    float* factors = (float*)(staging + PAIR_STAGING_BYTES);             // [group][half][block][row]
    uint64_t* full = (uint64_t*)(staging + PAIR_STAGING_BYTES + PAIR_FACTORS_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* fac_full = acc_empty + 2;
    uint64_t* fac_empty = fac_full + PAIR_GROUPS;
    uint32_t* tmem_slot = (uint32_t*)(fac_empty + PAIR_GROUPS);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    int* flag = error_word(p);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { init(&full[s], 1); init(&empty[s], 1); }
        for (int a = 0; a < 2; ++a) { init(&acc_full[a], 1); init(&acc_empty[a], 2 * PAIR_WARPS); }
        for (int g = 0; g < PAIR_GROUPS; ++g) { init(&fac_full[g], 2); init(&fac_empty[g], PAIR_WARPS); }
        fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(2 * PAIR_BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                  // the peer's barriers exist before anything signals them
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int a_tiles = p.a_tiles, b_tiles = (p.N + PAIR_BN - 1) / PAIR_BN;
    const int splits = p.splits, items = a_tiles * b_tiles * splits, first = blockIdx.x >> 1, stride = gridDim.x >> 1;
    // item i: part i % splits of the K of tile i / splits
    auto part_of_k = [&](int i, int& kb0, int& kb1) {
        kb0 = (int)((long long)p.kblocks * (i % splits) / splits);
        kb1 = (int)((long long)p.kblocks * (i % splits + 1) / splits);
    };

    pdl_launch_dependents();
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PAIR_REGS_LOW));
        if (threadIdx.x == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = first; i < items && ok; i += stride) {
                const int t = i / splits;
                int kb0, kb1;
                part_of_k(i, kb0, kb1);
                const int a0 = (t % a_tiles) * 2 * BM + (int)rank * BM, b0 = (t / a_tiles) * PAIR_BN + (int)rank * PAIR_HALF;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!wait(&empty[stage], phase ^ 1, flag, PH_ERR_FP8_PRODUCER)) { ok = false; break; }
                    const uint32_t bar = cluster_addr(&full[stage], 0);
                    // The leader alone announces the bytes of both; the peer's may land first (the count of bytes owed may run
                    // negative inside a phase, which still needs the leader's arrival).
                    if (leader) arrive_expect_tx(&full[stage], 2 * PAIR_STAGE_BYTES);
                    tma_load_2d_pair(smem_a + stage * A_BYTES, &map_a, bar, kb * BK, a0);
                    tma_load_2d_pair(smem_b + stage * PAIR_HALF * BK, &map_b, bar, kb * BK, b0);
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                }
            }
            // not past this point while copies may be in flight: the products have released every stage, or, after a wait that ran
            // out, the copies of both CTAs have at least arrived (the leader sees them; the peer waits for it at the end)
            for (int s = 0; s < STAGES; ++s) {
                if (ok && !wait(&empty[stage], phase ^ 1, flag, PH_ERR_FP8_PRODUCER)) ok = false;
                if (!ok && leader) wait(&full[stage], phase ^ 1, flag, PH_ERR_FP8_PRODUCER);
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
        } else if (threadIdx.x == 32 && leader) {
            constexpr uint32_t idesc = make_idesc(2 * BM, PAIR_BN);
            int stage = 0, buf = 0;
            uint32_t phase = 0, buf_phase = 0;
            bool ok = true;
            for (int i = first; i < items && ok; i += stride) {
                int kb0, kb1;
                part_of_k(i, kb0, kb1);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!wait(&full[stage], phase, flag, PH_ERR_FP8_MMA) || !wait(&acc_empty[buf], buf_phase ^ 1, flag, PH_ERR_FP8_MMA)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t adesc = smem_desc(smem_a + stage * A_BYTES), bdesc = smem_desc(smem_b + stage * PAIR_HALF * BK);
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)
                        umma_pair(tmem_base + (uint32_t)(buf * PAIR_BN), adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), idesc, k > 0 ? 1u : 0u);
                    umma_commit_pair(&acc_full[buf]);
                    umma_commit_pair(&empty[stage]);
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    if (++buf == 2) { buf = 0; buf_phase ^= 1; }
                }
            }
        } else if (warp >= 2) {
            // Two warps look the scales up, four blocks of K at a time and some groups ahead, and leave their products in shared memory:
            // 2048 x 9472 x 4096 takes 79 us, and 87 where the epilogue's threads load them for themselves, however far ahead.
            const int r = threadIdx.x - 64;
            int g = 0;
            uint32_t g_phase = 0;
            bool ok = true;
            for (int i = first; i < items && ok; i += stride) {
                const int t = i / splits;
                int kb0, kb1;
                part_of_k(i, kb0, kb1);
                const int row = (t % a_tiles) * 2 * BM + (int)rank * BM + r, nb = (t / a_tiles) * 2;
                const float* x0 = p.xs + (size_t)min(row, p.M - 1) * p.kblocks;
                const float* x1 = p.xs + (size_t)min(row + 64, p.M - 1) * p.kblocks;
                const float* w0 = p.ws + (size_t)nb * p.kblocks;
                const float* w1 = p.ws + (size_t)min(nb + 1, (p.N - 1) / BK) * p.kblocks;
                for (int kb = kb0; kb < kb1; kb += 4) {
                    float a[4], b[4], u[4], v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int k = min(kb + j, p.kblocks - 1);
                        a[j] = x0[k]; b[j] = x1[k]; u[j] = w0[k]; v[j] = w1[k];
                    }
                    ok = wait(&fac_empty[g], g_phase ^ 1, flag, PH_ERR_FP8_EPILOGUE);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    float* f = factors + g * 2 * 4 * BM + r;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[j * BM] = a[j] * u[j]; f[j * BM + 64] = b[j] * u[j];
                        f[(4 + j) * BM] = a[j] * v[j]; f[(4 + j) * BM + 64] = b[j] * v[j];
                    }
                    __syncwarp();
                    if (lane == 0) arrive(&fac_full[g]);
                    if (++g == PAIR_GROUPS) { g = 0; g_phase ^= 1; }
                }
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PAIR_REGS_HIGH));
        const int q = warp & 3, half = (warp - 4) >> 2;               // rows 32 q .. 32 q + 31, columns 128 half .. 128 half + 127
        uint8_t* boxes = staging + (warp - 4) * 2 * PAIR_BOX_BYTES;
        int turn = 0;
        int buf = 0;
        uint32_t buf_phase = 0;
        bool ok = true;
        int group = 0;
        uint32_t g_phase = 0;
        const uint32_t give_0 = cluster_addr(&acc_empty[0], 0), give_1 = cluster_addr(&acc_empty[1], 0);
        uint32_t taddr = 0;
        // this thread's factor of the item's block number b of `blocks` (each once, in order)
        auto next_factor = [&](int b, int blocks) {
            if ((b & 3) == 0) ok = ok && wait(&fac_full[group], g_phase, flag, PH_ERR_FP8_EPILOGUE);
            const float f = factors[((group * 2 + half) * 4 + (b & 3)) * BM + q * 32 + lane];
            if ((b & 3) == 3 || b + 1 == blocks) {
                __syncwarp();
                if (lane == 0) arrive(&fac_empty[group]);
                if (++group == PAIR_GROUPS) { group = 0; g_phase ^= 1; }
            }
            return f;
        };
        // waits for the next accumulator and asks for its first columns
        auto next_accumulator = [&](uint32_t* r) {
            ok = ok && wait(&acc_full[buf], buf_phase, flag, PH_ERR_FP8_EPILOGUE);
            __syncwarp();
            tc_fence_after();
            taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * PAIR_BN + half * PAIR_HALF);
            tmem_ld32(taddr, r);
        };
        for (int i = first; i < items; i += stride) {
            const int t = i / splits;
            int blocks, kb0;
            part_of_k(i, kb0, blocks);
            blocks -= kb0;
            const int row0 = (t % a_tiles) * 2 * BM + (int)rank * BM + q * 32, n0 = (t / a_tiles) * PAIR_BN + half * PAIR_HALF;
            float acc[PAIR_HALF];
#pragma unroll
            for (int j = 0; j < PAIR_HALF; ++j) acc[j] = 0.0f;
            // The loads run one chunk of 32 columns ahead of the multiply-adds, over the end of a block too, and so does the factor.
            uint32_t r[2][32];
            float f = next_factor(0, blocks), f_next = 0.0f;
            next_accumulator(r[0]);
#pragma unroll 1
            for (int b = 0; b < blocks; ++b) {
#pragma unroll
                for (int c = 0; c < PAIR_HALF / 32; ++c) {
                    tmem_ld_wait();
                    if (c + 1 < PAIR_HALF / 32) {
                        tmem_ld32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
                        if (c == 1 && b + 1 < blocks) f_next = next_factor(b + 1, blocks);
                    } else {
                        tc_fence_before();                            // all of it is in registers: the accumulator is free
                        __syncwarp();
                        if (lane == 0) arrive_cluster(buf ? give_1 : give_0);
                        if (++buf == 2) { buf = 0; buf_phase ^= 1; }
                        if (b + 1 < blocks) next_accumulator(r[0]);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 2) fma2(acc[c * 32 + j], acc[c * 32 + j + 1], r[c & 1][j], r[c & 1][j + 1], f);
                }
                f = f_next;
            }
            if (row0 >= p.M || (!GATED && n0 >= p.N)) continue;       // the whole warp (with the activation, both of a row's)
            if constexpr (GATED) {
                store_gated(p, acc, (float*)staging, turn, q, half, lane, row0 + lane, n0);
                turn ^= 1;
                continue;
            }
            // Boxes of 32 rows x 128 bytes, swizzled as the copy engine wants them (16-byte chunk ^ (row & 7)).  It stores them, and leaves
            // out what lies outside of out; rows that do not start on 16 bytes (an odd width) are stored by the warp, a row at a time
            // (3666 x 22705 x 432: 860 us where every thread stored its own row, value by value).
            const int n_boxes = p.out_bf16 ? 2 : 4;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (b >= n_boxes) break;
                uint8_t* box = boxes + (b & 1) * PAIR_BOX_BYTES;
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");       // this box of two has left
                __syncwarp();
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint4 v;
                    if (p.out_bf16) {
                        const float* a = acc + (b & 1) * 64 + c * 8;
                        v = make_uint4(bf16_pair(a[0], a[1]), bf16_pair(a[2], a[3]), bf16_pair(a[4], a[5]), bf16_pair(a[6], a[7]));
                    } else {
                        const float* a = acc + b * 32 + c * 4;
                        v = make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
                    }
                    *(uint4*)(box + lane * 128 + ((c ^ (lane & 7)) << 4)) = v;
                }
                const int col = n0 + b * (p.out_bf16 ? 64 : 32);
                if (p.tma_store) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if (col < p.N) tma_store_3d(&map_out, box, col, row0, i % splits);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");       // one group a box, stored or not: the count above goes by them
                    }
                } else {
                    __syncwarp();
                    const int rows = min(32, p.M - row0);
                    const size_t at = ((size_t)(i % splits) * p.M + row0) * p.N + col;
#pragma unroll 8
                    for (int r = 0; r < rows; ++r) {
                        const uint32_t v = *(const uint32_t*)(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                        if (p.out_bf16) {
                            uint16_t* o = (uint16_t*)p.out + at + (size_t)r * p.N + 2 * lane;
                            if (col + 2 * lane < p.N) o[0] = (uint16_t)v;
                            if (col + 2 * lane + 1 < p.N) o[1] = (uint16_t)(v >> 16);
                        } else if (col + lane < p.N) {
                            ((uint32_t*)p.out)[at + (size_t)r * p.N + lane] = v;
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                  // nothing of the peer may still reach this CTA
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * PAIR_BN) : "memory");
}

// ---- host side ---------------------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)f;
    });
    return fn;
}

// A [rows, K] matrix of bytes seen as boxes of box_rows x 128, 128-byte swizzle, zeros outside.
bool make_map(CUtensorMap* out, const void* ptr, int rows, int K, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)K};
    const cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// out [parts, rows, cols] seen as boxes of 32 rows x 128 bytes, 128-byte swizzle.
bool make_out_map(CUtensorMap* out, const void* ptr, bool bf16, int parts, int rows, int cols) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const int size = bf16 ? 2 : 4;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)parts};
    const cuuint64_t strides[2] = {(cuuint64_t)cols * size, (cuuint64_t)rows * cols * size};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / size), 32, 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    return fn(out, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(ptr), dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_pair(const void* x, const void* w, Params p, int K, cudaStream_t stream) {
    const bool gated = p.out_scales != nullptr;
    if (const int rc = gated ? allow_shared<gemm_fp8_pair_kernel<true>>(PAIR_SMEM_BYTES, "gemm_fp8_pair") : allow_shared<gemm_fp8_pair_kernel<false>>(PAIR_SMEM_BYTES, "gemm_fp8_pair")) return rc;
    CUtensorMap ma, mb, mo;
    if (!make_map(&ma, x, p.M, K, BM) || !make_map(&mb, w, p.N, K, PAIR_HALF))
        return fail(PH_ERR_LAUNCH, "gemm_fp8_pair: cuTensorMapEncodeTiled failed (M %d, N %d, K %d)", p.M, p.N, K);
    // the copy engine stores where its rules allow: rows of a multiple of 16 bytes on 16-byte boundaries
    mo = ma;
    p.tma_store = 0;
    if (!gated && (p.N * (p.out_bf16 ? 2LL : 4LL)) % 16 == 0 && ((uintptr_t)p.out & 15) == 0 && make_out_map(&mo, p.out, p.out_bf16, p.splits, p.M, p.N)) p.tma_store = 1;
    p.a_tiles = (p.M + 2 * BM - 1) / (2 * BM);
    const long long tiles = (long long)p.a_tiles * ((p.N + PAIR_BN - 1) / PAIR_BN) * p.splits;
    if (tiles > 0x3fffffffLL) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8_pair: %d x %d has too many tiles", p.M, p.N);
    const int clusters = (int)std::min<long long>(tiles, multiprocessors() / 2);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * clusters);
    cfg.blockDim = dim3(PAIR_THREADS);
    cfg.dynamicSmemBytes = PAIR_SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];                         // in plain stream order, as every cluster here
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, gated ? gemm_fp8_pair_kernel<true> : gemm_fp8_pair_kernel<false>, ma, mb, mo, p);
    return check_launch("gemm_fp8_pair");
}

template <int BN>
int launch(const void* x, const void* w, Params p, int K, cudaStream_t stream) {
    using Cfg = Tile<BN>;
    if (const int rc = allow_shared<gemm_fp8_kernel<BN>>(Cfg::SMEM_BYTES, "gemm_fp8")) return rc;
    CUtensorMap mw, mx;
    if (!make_map(&mw, w, p.N, K, BM) || !make_map(&mx, x, p.M, K, BN))
        return fail(PH_ERR_LAUNCH, "gemm_fp8: cuTensorMapEncodeTiled failed (M %d, N %d, K %d)", p.M, p.N, K);
    p.a_tiles = (p.N + BM - 1) / BM;
    const long long ctas = (long long)p.a_tiles * ((p.M + BN - 1) / BN) * p.splits;
    if (ctas > 0x7fffffffLL) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8: %d x %d has too many tiles", p.M, p.N);
    launch_overlapped(gemm_fp8_kernel<BN>, dim3((unsigned)ctas), dim3(THREADS), Cfg::SMEM_BYTES, stream, mw, mx, p);
    return check_launch("gemm_fp8");
}

// The tile (16, 32, 64 or 96 tokens beside 128 features; 256: pairs) and the parts of K with the least estimated time, among those that
// the caller leaves open (0).  Microseconds: a launch (a pair's does not start early), rounds of the CTAs over the device's places
// times (an item's start and end + its blocks of K), the weight's way from memory and the tiles' from L2, and for several parts
// their way out and back and the kernel that adds them up, or what they cost whoever consumes them.  Fitted to 1,538 launches at 1 to 2,048
// tokens, 256 to 24,576 features and K 512 to 16,384 (root mean square error 5 %); what it picks takes 1.5 % longer than the
// best of all, over those 80 products.  Tiles of 96 tokens, fitted to 327 more, are for 65 to 96 rows of wide weights: 72 x 24576 x 4096 takes
// 29 us in one, 38 in three of 32.  (Tiles of 128 tokens, with four epilogue warps, were never the best by more than 1 %; with eight and an
// SM for each CTA 128 x 24576 x 4096 took 40 us for 43, but 256 rows 64 for 44.  They are gone.)
// Parts that are handed on cost their consumer 0.8 us and 0.1 us each: with that, one row through the products, norms and
// quantizers of a layer of the 8B shape takes 46.5 us and not 48.3 (gate and up whole, not in three parts).
void choose(int M, int N, int K, int sms, bool whole, int* tile, int* splits) {
    struct Kind { int tile, per_sm; double launch, item, block; };
    static const Kind kinds[] = {{16, 2, 0.26, 1.92, 0.339}, {32, 2, 0.26, 2.34, 0.358}, {64, 2, 0.26, 3.61, 0.404}, {96, 2, 0.26, 4.84, 0.54}, {256, 0, 4.08, 1.54, 0.491}};
    const int kblocks = (K + BK - 1) / BK, asked_tile = *tile, asked_splits = *splits;
    const double weight_mb = 1e-6 * N * K;
    double best = -1.0;
    for (const Kind& k : kinds) {
        if (asked_tile != 0 && k.tile != asked_tile) continue;
        const bool pair = k.tile == 256;
        const double tiles = (double)((N + (pair ? 255 : 127)) / (pair ? 256 : 128)) * ((M + k.tile - 1) / k.tile);
        const double slots = pair ? sms / 2 : sms * k.per_sm, stage_mb = 1e-6 * BK * (pair ? 512 : 128 + k.tile);
        for (int s = 1; s <= MAX_SPLITS && s <= kblocks; ++s) {
            if (asked_splits != 0 && s != asked_splits) continue;
            const int blocks = (kblocks + s - 1) / s;
            double cost = k.launch + ceil(tiles * s / slots) * (k.item + k.block * blocks) + weight_mb / 28.2 + tiles * s * blocks * stage_mb / 51.7;
            if (s > 1) cost += (whole ? 1.38 + 0.136 * s : 0.8 + 0.236 * s) + s * 8e-6 * M * N / 9.8;
            if (best < 0 || cost < best - 1e-9) { best = cost; *tile = k.tile; *splits = s; }
        }
    }
}

}  // namespace

// How ph_gemm_fp8 should cut an M x N x K product on the current device: *tile and *splits where they are 0 (the other one may be
// given).  whole: the whole sum is wanted, not the parts.
PH_EXPORT int ph_gemm_fp8_plan(int M, int N, int K, int whole, int* tile, int* splits) {
    if (M < 1 || N < 1 || K < 1 || M > MAX_SIZE || N > MAX_SIZE || K > MAX_SIZE || !tile || !splits || *tile < 0 || *splits < 0) return fail(PH_ERR_ARG, "gemm_fp8: no plan for M %d, N %d, K %d", M, N, K);
    const int kblocks = (K + BK - 1) / BK;
    if (*tile != 0 && *tile != 16 && *tile != 32 && *tile != 64 && *tile != 96 && *tile != 256) return fail(PH_ERR_ARG, "gemm_fp8: tile %d is not one of 16, 32, 64, 96, 256", *tile);
    if (*splits > kblocks || *splits > MAX_SPLITS) return fail(PH_ERR_ARG, "gemm_fp8: %d parts of K for %d blocks (at most %d)", *splits, kblocks, MAX_SPLITS);
    choose(M, N, K, multiprocessors(), whole != 0, tile, splits);
    return PH_OK;
}

// out = x times w transposed, with scales (above); xs [M, ceil(K / 128)], ws [ceil(N / 128), ceil(K / 128)].  tile: 16, 32, 64 or 96 tokens
// beside 128 features, or 256: 256 x 256 on pairs of CTAs.  splits: parts of K, 1 to 16.  With several, parts is room for
// [splits][M, N] float32: the sums of each part go there, and then, where out is given, their sum to out.  With one, or for the sum,
// out [M, N] is float32 or bfloat16.  early_w: w and ws are not results of a kernel that may still run when this one starts, and the first
// tiles of w may be read before the kernel in front has ended.  error_flag: where a wait that ran out leaves its number (null: see
// ph_fp8_take_error).
PH_EXPORT int ph_gemm_fp8(const void* x, const float* xs, const void* w, const float* ws, void* out, int out_dtype, int M, int N, int K, int tile,
                          int splits, float* parts, int early_w, int* error_flag, cudaStream_t stream) {
    if (M == 0) return PH_OK;
    if (!x || !xs || !w || !ws || M < 1 || N < 1 || K < 1 || !valid_dtype(out_dtype)) return fail(PH_ERR_ARG, "gemm_fp8: bad arguments (M %d, N %d, K %d)", M, N, K);
    if (M > MAX_SIZE || N > MAX_SIZE || K > MAX_SIZE) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8: M, N and K of at most %d, not %d, %d and %d", MAX_SIZE, M, N, K);
    if (K % 16) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8: K = %d must be a multiple of 16 (16-byte rows for TMA)", K);
    if (((uintptr_t)x | (uintptr_t)w) & 15) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8: operands must be 16-byte aligned");
    Params p = {};
    p.xs = xs; p.ws = ws; p.M = M; p.N = N; p.kblocks = (K + BK - 1) / BK; p.splits = splits; p.early_w = early_w; p.error_flag = error_flag;
    if (splits < 1 || splits > MAX_SPLITS || splits > p.kblocks) return fail(PH_ERR_ARG, "gemm_fp8: %d parts of K for %d blocks (at most %d)", splits, p.kblocks, MAX_SPLITS);
    if (splits == 1 ? !out : !parts) return fail(PH_ERR_ARG, "gemm_fp8: no room for the result");
    if (splits > 1 && out && ((uintptr_t)parts & 15)) return fail(PH_ERR_ARG, "gemm_fp8: parts that are summed here must be 16-byte aligned");
    p.out = splits > 1 ? parts : out;
    p.out_bf16 = splits == 1 && out_dtype == PH_BF16;
    int rc;
    switch (tile) {
        case 16: rc = launch<16>(x, w, p, K, stream); break;
        case 32: rc = launch<32>(x, w, p, K, stream); break;
        case 64: rc = launch<64>(x, w, p, K, stream); break;
        case 96: rc = launch<96>(x, w, p, K, stream); break;
        case 256:
            rc = launch_pair(x, w, p, K, stream);
            break;
        default: return fail(PH_ERR_ARG, "gemm_fp8: tile %d is not one of 16, 32, 64, 96, 256", tile);
    }
    if (rc != PH_OK || splits == 1 || !out) return rc;
    const long long values = (long long)M * N, grid = (values + 1023) / 1024;
    if (grid > 0x7fffffffLL) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8: %d x %d is too much", M, N);
    if (out_dtype == PH_BF16) launch_overlapped(sum_parts_kernel<__nv_bfloat16>, dim3((unsigned)grid), dim3(256), 0, stream, (const float*)parts, splits, values, (__nv_bfloat16*)out);
    else launch_overlapped(sum_parts_kernel<float>, dim3((unsigned)grid), dim3(256), 0, stream, (const float*)parts, splits, values, (float*)out);
    return check_launch("gemm_fp8 (sum of the parts)");
}

// The product of (gate, up) rows with the gated activation behind it, in 8 bits: w [N, K] holds the rows of gate and up in turn, q [M, N / 2] and
// scales [M, N / 256] what ph_gated_fp8 would make of the float32 product (which never leaves the SMs).  On pairs of CTAs, K whole; N a multiple of 256.
// gate: as ph_gated_fp8's.
PH_EXPORT int ph_gemm_fp8_gated(const void* x, const float* xs, const void* w, const float* ws, void* q, float* scales, int M, int N, int K, const float* gate, int* error_flag,
                                cudaStream_t stream) {
    if (M == 0) return PH_OK;
    if (!x || !xs || !w || !ws || !q || !scales || M < 1 || N < 1 || K < 1) return fail(PH_ERR_ARG, "gemm_fp8_gated: bad arguments (M %d, N %d, K %d)", M, N, K);
    if (M > MAX_SIZE || N > MAX_SIZE || K > MAX_SIZE) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8_gated: M, N and K of at most %d, not %d, %d and %d", MAX_SIZE, M, N, K);
    if (K % 16 || N % PAIR_BN) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8_gated: K = %d must be a multiple of 16 and N = %d one of %d", K, N, PAIR_BN);
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)q) & 15) return fail(PH_ERR_UNSUPPORTED, "gemm_fp8_gated: operands and q must be 16-byte aligned");
    Params p = {};
    p.xs = xs; p.ws = ws; p.M = M; p.N = N; p.kblocks = (K + BK - 1) / BK; p.splits = 1; p.error_flag = error_flag; p.out = q; p.out_scales = scales;
    p.gate = ph_fp8::Gate{0, 1.0f, 0.0f, 0.0f};
    if (gate) p.gate = ph_fp8::Gate{(int)gate[3], gate[0], gate[1], gate[2]};
    if (p.gate.kind < 0 || p.gate.kind > 2) return fail(PH_ERR_ARG, "gemm_fp8_gated: gate %d is not known", p.gate.kind);
    return launch_pair(x, w, p, K, stream);
}

// The number that a wait which ran out has left on the current device since the last call (0: none); waits for the device.
PH_EXPORT int ph_fp8_take_error(int* code) {
    if (!code) return fail(PH_ERR_ARG, "fp8_take_error: no place for the number");
    const int zero = 0;
    if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(code, g_error, sizeof(int)) != cudaSuccess ||
        (*code != 0 && cudaMemcpyToSymbol(g_error, &zero, sizeof(int)) != cudaSuccess))
        return fail(PH_ERR_LAUNCH, "fp8_take_error: %s", cudaGetErrorString(cudaGetLastError()));
    return PH_OK;
}
