// Rows and weights in 8 bits (e4m3) with a float32 scale for each block, and the two passes that give such rows: the
// norm behind the residual's addition, and the gated activation.
//
// A block is 128 values of a row (the last one of a row may be shorter), or 128 x 128 values of a weight.  With amax the
// block's largest magnitude and a = max(amax, 448 * 2^-126): scale = a / 448, q = e4m3(x * (448 / a)), rounded to nearest,
// ties to even.  The lower bound keeps both quotients finite for blocks of zeros and of the smallest numbers; a value that is
// no number makes its block's scale and values none, an infinite one makes the scale infinite, so that neither is lost.
// Everything in front of the rounding to 8 bits is float32.
//
// Half a warp owns a block of a row: 16 lanes of 8 values, read as 16-byte vectors (two for float32) and written as 8 bytes
// a lane, the largest magnitude found by four exchanges.  Where rows do not lie on such boundaries (a width that is no multiple of
// eight, a stride or a base that is no multiple of 16 bytes) a lane takes every 16th pair of values instead, or, where a pair does
// not lie on its own boundary either (an odd width), every 16th value.  All three passes are bound by
// memory: each input is read once and held in registers until its block's scale is known.
// The reference's counterpart is its 8-bit activation blocks (src/matvec_q.hip), whose scales are per 32 values.
#include "common.cuh"
#include "fp8_values.cuh"
#include "shared_limit.cuh"

namespace {

using namespace ph;
using namespace ph_fp8;

constexpr int MAX_WIDTH = 1 << 30;                             // of a row: its blocks are counted in 32 bits
// The largest magnitude over the 16 lanes that share a block.
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The place of a lane's value i inside its block, for vectors of W values.
template <int W> __device__ __forceinline__ int place(int lane16, int i) {
    return W == 8 ? lane16 * 8 + i : W == 2 ? 32 * (i >> 1) + lane16 * 2 + (i & 1) : lane16 + 16 * i;
}

// A lane's eight values of a block as they lie in memory, and what is asked of them: a bfloat16 block waits for its scale in
// half the registers, and its largest magnitude is found two values at a time.
template <typename T> struct Held;
template <> struct Held<float> {
    float v[8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
    __device__ __forceinline__ void load(const float* p) { load8(p, v); }
    __device__ __forceinline__ void load2(int i, const float* p) {                      // values 2 i and 2 i + 1
        const float2 u = *reinterpret_cast<const float2*>(p);
        v[2 * i] = u.x; v[2 * i + 1] = u.y;
    }
    __device__ __forceinline__ void load4(int i, const float* p) {                      // values 4 i .. 4 i + 3
        const float4 u = *reinterpret_cast<const float4*>(p);
        v[4 * i] = u.x; v[4 * i + 1] = u.y; v[4 * i + 2] = u.z; v[4 * i + 3] = u.w;
    }
    __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
    __device__ __forceinline__ float get(int i) const { return v[i]; }
    __device__ __forceinline__ float largest() const {
        float m = fabsf(v[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
        return m;
    }
};
template <> struct Held<__nv_bfloat16> {
    uint32_t v[4];
    __device__ __forceinline__ void clear() { v[0] = v[1] = v[2] = v[3] = 0; }
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
    __device__ __forceinline__ void load2(int i, const __nv_bfloat16* p) { v[i] = *reinterpret_cast<const uint32_t*>(p); }
    __device__ __forceinline__ void load4(int i, const __nv_bfloat16* p) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        v[2 * i] = u.x; v[2 * i + 1] = u.y;
    }
    __device__ __forceinline__ void set(int i, __nv_bfloat16 x) {
        const uint32_t bits = __bfloat16_as_ushort(x);
        v[i >> 1] = (i & 1) ? (v[i >> 1] & 0xffffu) | bits << 16 : (v[i >> 1] & 0xffff0000u) | bits;
    }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float((i & 1) ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16); }
    __device__ __forceinline__ float largest() const {
        __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v[0]));
#pragma unroll
        for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v[i])));
        return max_nan(__low2float(m), __high2float(m));
    }
};

// A lane's eight values of the block that starts at column k0 of a row of K (zeros behind the row's end).
template <int W, typename T>
__device__ __forceinline__ void hold_block(const T* row, int k0, int lane16, int K, Held<T>& h) {
    h.clear();
    if (W == 8) {
        if (k0 + lane16 * 8 < K) h.load(row + k0 + lane16 * 8);
    } else if (W == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + place<2>(lane16, 2 * i);
            if (k < K) h.load2(i, row + k);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = k0 + place<1>(lane16, i);
            if (k < K) h.set(i, row[k]);
        }
    }
}
template <int W, typename T>
__device__ __forceinline__ void load_block(const T* row, int k0, int lane16, int K, float* v) {
    Held<T> h;
    hold_block<W>(row, k0, lane16, K, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = h.get(i);
}

template <int W, typename V>
__device__ __forceinline__ void store_block(uint8_t* row, int k0, int lane16, int K, const V& v, float inverse) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = pack2(v.get(2 * i) * inverse, v.get(2 * i + 1) * inverse);
    if (W == 8) {
        if (k0 + lane16 * 8 < K) *(uint2*)(row + k0 + lane16 * 8) = make_uint2(p[0] | p[1] << 16, p[2] | p[3] << 16);
    } else if (W == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + place<2>(lane16, 2 * i);
            if (k < K) *(uint16_t*)(row + k) = (uint16_t)p[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = k0 + place<1>(lane16, i);
            if (k < K) row[k] = (uint8_t)(p[i >> 1] >> (8 * (i & 1)));
        }
    }
}

// A lane's share of a block: the block's scale to *scale, its values to the row.  Every lane of the warp calls this.
template <int W, typename V>
__device__ __forceinline__ void finish_block(uint8_t* row, float* scale, bool live, int k0, int lane16, int K, const V& v) {
    const float a = max_nan(half_warp_max(v.largest()), LEAST);
    if (!live) return;
    if (lane16 == 0) *scale = a / TOP;
    store_block<W>(row, k0, lane16, K, v, TOP / a);
}

constexpr int ROW_THREADS = 128;      // (2,048 rows of 12,288 gated values: 23.2 us; CTAs of 256 threads 24.0, of 512 27.3, of 64 23.1, but few rows 25 % longer)

// U neighbouring blocks of rows for each half warp, all of them asked for before the first is worked on.
template <typename T, int W, int U>
__global__ void __launch_bounds__(ROW_THREADS) quantize_rows_kernel(const T* __restrict__ x, long long stride, uint8_t* __restrict__ q, float* __restrict__ scales, unsigned blocks,
                                     unsigned kblocks, int K) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane16 = threadIdx.x & 15;
    const unsigned first = (blockIdx.x * (ROW_THREADS / 16) + (threadIdx.x >> 4)) * U;
    unsigned row = first / kblocks, b = first - row * kblocks;
    Held<T> v[U];
    unsigned at_row[U];
    int k0[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        at_row[u] = row;
        k0[u] = (int)b * BLOCK;
        if (first + u < blocks) hold_block<W>(x + row * stride, k0[u], lane16, K, v[u]);
        else v[u].clear();
        if (++b == kblocks) { b = 0; ++row; }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        finish_block<W>(q + (size_t)at_row[u] * K, scales + first + u, first + u < blocks, k0[u], lane16, K, v[u]);
}

// One CTA for each 128 x 128 block of a weight: 16 half warps, eight rows each.
template <typename T, int W>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const T* __restrict__ x, long long stride, uint8_t* __restrict__ q, float* __restrict__ scales, int T_rows, int K) {
    __shared__ float part[8];
    pdl_wait();
    const int lane16 = threadIdx.x & 15, half = threadIdx.x >> 4;
    const int k0 = blockIdx.x * BLOCK;
    const long long t0 = (long long)blockIdx.y * BLOCK;
    Held<T> v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const long long t = t0 + r * 16 + half;
        if (t < T_rows) hold_block<W>(x + t * stride, k0, lane16, K, v[r]);
        else v[r].clear();
    }
    float m = v[0].largest();
#pragma unroll
    for (int r = 1; r < 8; ++r) m = max_nan(m, v[r].largest());
    m = half_warp_max(m);
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max_nan(m, part[w]);
    const float a = max_nan(m, LEAST);
    if (threadIdx.x == 0) scales[(long long)blockIdx.y * gridDim.x + blockIdx.x] = a / TOP;
    const float inverse = TOP / a;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const long long t = t0 + r * 16 + half;
        if (t < T_rows) store_block<W>(q + t * K, k0, lane16, K, v[r], inverse);
    }
}

// v = x[t] + sum over the parts of add[s][t]; v to x_out[t] (or nowhere); y = v * rsqrt(mean(v^2) + eps) * weight to 8 bits.
// One CTA a row, U blocks for each half warp.  AHEAD: how many parts are asked for at a time (they are added in their order); above 1
// the weight comes before the row's sum too, and a line of it to L2 before the kernel in front is done.  (CTAs that walk over the rows,
// the next ones on their way to shared memory meanwhile, took 35 us for 2,048 rows of 5,120 where one CTA a row takes 23: their two
// barriers a row are then in one another's way.)
constexpr int ALONE = 6;             // the AHEAD of CTAs that have an SM for themselves, in the registers that this leaves
struct NormParams {
    const float* x;
    const void* add;
    int parts;
    long long part_stride;
    const float* weight;
    float eps;
    const int32_t* rows;         // row r of the output is row rows[r] of the input (null: r); a row outside 0 .. T - 1 is left out
    int T, E, kblocks;
    float* x_out;
    uint8_t* q;
    float* scales;
};

template <typename A, int W, int U, int AHEAD>
__global__ void __launch_bounds__(AHEAD == ALONE ? 640 : 1024) add_rmsnorm_fp8_kernel(NormParams p) {
    constexpr bool MORE = AHEAD > 1;
    __shared__ float scratch[32];
    const int lane16 = threadIdx.x & 15, half = threadIdx.x >> 4, halves = blockDim.x >> 4;
    pdl_launch_dependents();
#pragma unroll
    for (int u = 0; u < (MORE ? U : 0); ++u) {
        const int k = (half + u * halves) * BLOCK + lane16 * 8;
        if (k < p.E) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.weight + k));
    }
    pdl_wait();
    const long long r = blockIdx.x;
    const long long t = p.rows ? p.rows[r] : r;
    if (t < 0 || t >= p.T) return;                     // the whole CTA
    const float* x = p.x + t * p.E;
    const A* add = (const A*)p.add + t * p.E;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) load_block<W>(x, (half + u * halves) * BLOCK, lane16, p.E, v[u]);
    if (p.add) {
        for (int s = 0; s < p.parts; s += AHEAD) {
            Held<A> a[AHEAD][U];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s + j < p.parts) hold_block<W>(add + (s + j) * p.part_stride, (half + u * halves) * BLOCK, lane16, p.E, a[j][u]);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (s + j < p.parts) v[u][i] += a[j][u].get(i);
        }
    }
    float w[U][8];
    if (MORE) {
#pragma unroll
        for (int u = 0; u < U; ++u) load_block<W>(p.weight, (half + u * halves) * BLOCK, lane16, p.E, w[u]);
    }
    float ss = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += v[u][i] * v[u][i];
    if (p.x_out) {
        float* o = p.x_out + t * p.E;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = (half + u * halves) * BLOCK;
            if (W == 8) {
                if (k0 + lane16 * 8 < p.E) store8(o + k0 + lane16 * 8, v[u]);
            } else if (W == 2) {
#pragma unroll
                for (int i = 0; i < 8; i += 2)
                    if (k0 + place<2>(lane16, i) < p.E) *(float2*)(o + k0 + place<2>(lane16, i)) = make_float2(v[u][i], v[u][i + 1]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + place<1>(lane16, i) < p.E) o[k0 + place<1>(lane16, i)] = v[u][i];
            }
        }
    }
    const float f = rsqrtf(block_sum_any(ss, scratch) / (float)p.E + p.eps);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int b = half + u * halves;
        if (!MORE) load_block<W>(p.weight, b * BLOCK, lane16, p.E, w[u]);
        Held<float> y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y.v[i] = v[u][i] * f * w[u][i];
        finish_block<W>(p.q + r * p.E, p.scales + r * p.kblocks + b, b < p.kblocks, b * BLOCK, lane16, p.E, y);
    }
}

// Rows of (g0, u0, g1, u1, ...), in `parts` parts that are summed first, to gated rows of F in 8 bits; U blocks for each half warp.
template <typename T, int W, int U>
__global__ void __launch_bounds__(ROW_THREADS) gated_fp8_kernel(const T* __restrict__ gate_up, int parts, long long part_stride, uint8_t* __restrict__ q, float* __restrict__ scales,
                                 unsigned blocks, unsigned kblocks, int F, Gate gate) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane16 = threadIdx.x & 15;
    const unsigned first = (blockIdx.x * (ROW_THREADS / 16) + (threadIdx.x >> 4)) * U;
    unsigned row = first / kblocks, b = first - row * kblocks;
    const bool pairs = ((uintptr_t)gate_up & (2 * sizeof(T) - 1)) == 0;       // (a pair never straddles its own boundary then)
    if (parts == 1) {
        // one part: what is read waits as it lies in memory
        Held<T> v[U][2];
        unsigned at_row[U];
        int k0[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at_row[u] = row;
            k0[u] = (int)b * BLOCK;
            v[u][0].clear();
            v[u][1].clear();
            const T* src = gate_up + (size_t)row * 2 * F;
            if (first + u >= blocks) {
            } else if (W == 8) {
                if (k0[u] + lane16 * 8 < F) {
                    v[u][0].load(src + 2 * (k0[u] + lane16 * 8));
                    v[u][1].load(src + 2 * (k0[u] + lane16 * 8) + 8);
                }
            } else if (W == 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = k0[u] + place<2>(lane16, 2 * i);
                    if (k < F) v[u][i >> 1].load4(i & 1, src + 2 * (size_t)k);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = k0[u] + place<1>(lane16, i);
                    if (k >= F) continue;
                    if (pairs) v[u][i >> 2].load2(i & 3, src + 2 * (size_t)k);
                    else {
                        v[u][i >> 2].set(2 * (i & 3), src[2 * (size_t)k]);
                        v[u][i >> 2].set(2 * (i & 3) + 1, src[2 * (size_t)k + 1]);
                    }
                }
            }
            if (++b == kblocks) { b = 0; ++row; }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Held<float> h;
#pragma unroll
            for (int i = 0; i < 8; ++i) h.v[i] = gated_value(gate, v[u][i >> 2].get(2 * (i & 3)), v[u][i >> 2].get(2 * (i & 3) + 1));
            finish_block<W>(q + (size_t)at_row[u] * F, scales + first + u, first + u < blocks, k0[u], lane16, F, h);
        }
        return;
    }
#pragma unroll 1
    for (int u = 0; u < U; ++u) {
        const int k0 = (int)b * BLOCK;
        const bool live = first + u < blocks;
        const T* src = gate_up + (size_t)row * 2 * F;
        Held<float> h;
        if (W == 8) {
            float g[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) g[i] = 0.0f;
            if (live && k0 + lane16 * 8 < F) {
                for (int s = 0; s < parts; s += 3) {                 // three at a time (8 rows of 12,288: 2.1 us, 2.2 one by one; 64 4.1 and 4.6)
                    Held<T> a[3][2];
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        if (s + j < parts) {
                            a[j][0].load(src + (s + j) * part_stride + 2 * (k0 + lane16 * 8));
                            a[j][1].load(src + (s + j) * part_stride + 2 * (k0 + lane16 * 8) + 8);
                        }
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        if (s + j < parts) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) g[i] = s + j == 0 ? a[j][i >> 3].get(i & 7) : g[i] + a[j][i >> 3].get(i & 7);
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) h.v[i] = gated_value(gate, g[2 * i], g[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = k0 + place<W>(lane16, i);
                float g = 0.0f, x = 0.0f;
                if (live && k < F) {
                    g = to_float<T>(src[2 * (size_t)k]); x = to_float<T>(src[2 * (size_t)k + 1]);
                    for (int s = 1; s < parts; ++s) { g += to_float<T>(src[s * part_stride + 2 * (size_t)k]); x += to_float<T>(src[s * part_stride + 2 * (size_t)k + 1]); }
                }
                h.v[i] = gated_value(gate, g, x);
            }
        }
        finish_block<W>(q + (size_t)row * F, scales + first + u, live, k0, lane16, F, h);
        if (++b == kblocks) { b = 0; ++row; }
    }
}

// Blocks for each half warp where they are many: what a lane holds while it waits is the same for both types.
template <typename T> constexpr int MANY = 8 / (int)sizeof(T);

// The number of blocks and of CTAs for them.  Several blocks a half warp once every SM has 256 blocks, else one: 2,048 rows of
// 12,288 gated bfloat16 values take 23.2 us with four, 25.2 with two and 34.7 with eight (and 26.7 where as many CTAs as the device
// holds walk over the blocks); 256 such rows 6.5 with four and 5.5 with one.
inline bool count_blocks(long long rows, int width, int many, unsigned* blocks, int* u, unsigned* ctas) {
    const long long n = rows * ((width + BLOCK - 1) / BLOCK);
    if (n > 0x7fffffffLL - 4 * ROW_THREADS) return false;
    *blocks = (unsigned)n;
    *u = n >= (long long)multiprocessors() * 256 ? many : 1;
    *ctas = (unsigned)((n + (ROW_THREADS / 16) * *u - 1) / ((ROW_THREADS / 16) * *u));
    return true;
}

inline bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

template <typename A, int W>
int launch_norm(const NormParams& p, int n, cudaStream_t stream) {
    // blocks per half warp: as few as a CTA of 1,024 threads allows, so that a row is spread wide and waits for its sum the
    // shortest (2,048 rows of 5,120: 20.5 us with one, 24.5 with two, 29.8 with four)
    const int u = p.kblocks <= 64 ? 1 : p.kblocks <= 128 ? 2 : 4;
    const int halves = (p.kblocks + u - 1) / u;
    const int threads = (halves * 16 + 31) / 32 * 32;
    // Several parts come from few rows: one request behind the other, a row of 4,096 in nine of them took 3.7 us, four at a time 3.3.  Where
    // every row has an SM for itself six are asked for (in a layer of an 8B shape behind its products, two norms of 64 rows 9.5 us with
    // four, 6.0 with six); 300 rows of three parts take 7.3 us with four and 8.6 with six.
    auto kernel = u == 4 ? add_rmsnorm_fp8_kernel<A, W, 4, 1> : u == 2 ? (p.parts > 1 ? add_rmsnorm_fp8_kernel<A, W, 2, 2> : add_rmsnorm_fp8_kernel<A, W, 2, 1>)
                : p.parts == 1 ? add_rmsnorm_fp8_kernel<A, W, 1, 1> : threads <= 640 && n <= multiprocessors() ? add_rmsnorm_fp8_kernel<A, W, 1, ALONE> : add_rmsnorm_fp8_kernel<A, W, 1, 4>;
    launch_overlapped(kernel, dim3(n), dim3(threads), 0, stream, p);
    return check_launch("add_rmsnorm_fp8");
}

}  // namespace

// x [T, K] in rows of `stride` elements to q [T, K] and scales [ceil(T / block_rows), ceil(K / 128)]; block_rows 1 or 128.
PH_EXPORT int ph_quantize_fp8(const void* x, int dtype, long long stride, void* q, float* scales, int T, int K, int block_rows, cudaStream_t stream) {
    if (T == 0) return PH_OK;
    if (!x || !q || !scales || T < 0 || K < 1 || stride < K || !valid_dtype(dtype)) return fail(PH_ERR_ARG, "quantize_fp8: bad arguments (T %d, K %d, row stride %lld)", T, K, stride);
    if (K > MAX_WIDTH) return fail(PH_ERR_UNSUPPORTED, "quantize_fp8: rows of at most %d values, not %d", MAX_WIDTH, K);
    if (block_rows != 1 && block_rows != BLOCK) return fail(PH_ERR_ARG, "quantize_fp8: blocks are of 1 or 128 rows, not %d", block_rows);
    const int kblocks = (K + BLOCK - 1) / BLOCK;
    const int size = dtype == PH_F32 ? 4 : 2;
    const int w = K % 8 == 0 && (stride * size) % 16 == 0 && aligned(x, 16) && aligned(q, 8) ? 8 : K % 2 == 0 && stride % 2 == 0 && aligned(x, 2 * size) && aligned(q, 2) ? 2 : 1;
    if (block_rows == BLOCK) {
        if (T > 65535 * BLOCK) return fail(PH_ERR_UNSUPPORTED, "quantize_fp8: a weight of at most 65535 * 128 rows, not %d", T);
        const dim3 grid(kblocks, (T + BLOCK - 1) / BLOCK);
        PH_DISPATCH(dtype, X, {
            auto kernel = w == 8 ? quantize_blocks_kernel<X, 8> : w == 2 ? quantize_blocks_kernel<X, 2> : quantize_blocks_kernel<X, 1>;
            launch_overlapped(kernel, grid, dim3(256), 0, stream, (const X*)x, stride, (uint8_t*)q, scales, T, K);
        });
        return check_launch("quantize_fp8");
    }
    const int many = dtype == PH_F32 ? MANY<float> : MANY<__nv_bfloat16>;
    unsigned blocks, ctas;
    int u;
    if (!count_blocks(T, K, many, &blocks, &u, &ctas)) return fail(PH_ERR_UNSUPPORTED, "quantize_fp8: %d x %d are too many blocks", T, K);
    PH_DISPATCH(dtype, X, {
        auto kernel = w == 8 ? (u == 1 ? quantize_rows_kernel<X, 8, 1> : quantize_rows_kernel<X, 8, MANY<X>>)
                    : w == 2 ? (u == 1 ? quantize_rows_kernel<X, 2, 1> : quantize_rows_kernel<X, 2, MANY<X>>)
                             : (u == 1 ? quantize_rows_kernel<X, 1, 1> : quantize_rows_kernel<X, 1, MANY<X>>);
        launch_overlapped(kernel, dim3(ctas), dim3(ROW_THREADS), 0, stream, (const X*)x, stride, (uint8_t*)q, scales, blocks, (unsigned)kblocks, K);
    });
    return check_launch("quantize_fp8");
}

// x [T, E] float32 += the parts of add ([parts][T, E], part_stride elements apart; null: nothing), kept in x_out [T, E] (x itself, another
// array or null); the normed rows to q [n, E] and scales [n, ceil(E / 128)].  rows [n] (or null): which rows, in that order.
PH_EXPORT int ph_add_rmsnorm_fp8(const float* x, const void* add, int add_dtype, int parts, long long part_stride, const float* weight, float eps,
                                 const int32_t* rows, int n, int T, int E, float* x_out, void* q, float* scales, cudaStream_t stream) {
    if (n == 0) return PH_OK;
    if (!x || !weight || !q || !scales || n < 0 || T < 1 || E < 1 || parts < 1 || !valid_dtype(add_dtype) || !(eps >= 0.0f))
        return fail(PH_ERR_ARG, "add_rmsnorm_fp8: bad arguments (T %d, E %d, rows %d, parts %d, eps %g)", T, E, n, parts, (double)eps);
    if (rows && x_out) return fail(PH_ERR_ARG, "add_rmsnorm_fp8: the sums of picked rows are not kept");
    const int kblocks = (E + BLOCK - 1) / BLOCK;
    if (kblocks > 256) return fail(PH_ERR_UNSUPPORTED, "add_rmsnorm_fp8: rows of at most 32768 values, not %d", E);
    NormParams p = {x, add, parts, part_stride, weight, eps, rows, T, E, kblocks, x_out, (uint8_t*)q, scales};
    const int size = add_dtype == PH_F32 ? 4 : 2;
    const bool v8 = E % 8 == 0 && aligned(x, 16) && aligned(weight, 16) && aligned(x_out, 16) && aligned(q, 8) && aligned(add, 16) && (part_stride * size) % 16 == 0;
    const bool v2 = E % 2 == 0 && aligned(x, 8) && aligned(weight, 8) && aligned(x_out, 8) && aligned(q, 2) && aligned(add, 2 * size) && part_stride % 2 == 0;
    PH_DISPATCH(add_dtype, A, { return v8 ? launch_norm<A, 8>(p, n, stream) : v2 ? launch_norm<A, 2>(p, n, stream) : launch_norm<A, 1>(p, n, stream); });
}

// gate_up [parts][T, 2 F] (part_stride elements apart) of (gate, up) pairs to q [T, F] and scales [T, ceil(F / 128)].  gate: null
// (silu), or four floats on the host: alpha, limit, shift and the kind (1 clamped swish, 2 the tanh form of gelu).
PH_EXPORT int ph_gated_fp8(const void* gate_up, int dtype, int parts, long long part_stride, void* q, float* scales, int T, int F, const float* gate,
                           cudaStream_t stream) {
    if (T == 0) return PH_OK;
    if (!gate_up || !q || !scales || T < 0 || F < 1 || F > 0x3fffffff || parts < 1 || !valid_dtype(dtype)) return fail(PH_ERR_ARG, "gated_fp8: bad arguments (T %d, F %d, parts %d)", T, F, parts);
    Gate g = {0, 1.0f, 0.0f, 0.0f};
    if (gate) g = Gate{(int)gate[3], gate[0], gate[1], gate[2]};
    if (g.kind < 0 || g.kind > 2) return fail(PH_ERR_ARG, "gated_fp8: gate %d is not known", g.kind);
    const int kblocks = (F + BLOCK - 1) / BLOCK, size = dtype == PH_F32 ? 4 : 2;
    const int many = dtype == PH_F32 ? MANY<float> : MANY<__nv_bfloat16>;
    unsigned blocks, ctas;
    int u;
    if (!count_blocks(T, F, many, &blocks, &u, &ctas)) return fail(PH_ERR_UNSUPPORTED, "gated_fp8: %d x %d are too many blocks", T, F);
    const int w = F % 8 == 0 && aligned(gate_up, 16) && aligned(q, 8) && (part_stride * size) % 16 == 0 ? 8 : F % 2 == 0 && aligned(gate_up, 4 * size) && aligned(q, 2) ? 2 : 1;
    PH_DISPATCH(dtype, X, {
        auto kernel = w == 8 ? (u == 1 ? gated_fp8_kernel<X, 8, 1> : gated_fp8_kernel<X, 8, MANY<X>>)
                    : w == 2 ? (u == 1 ? gated_fp8_kernel<X, 2, 1> : gated_fp8_kernel<X, 2, MANY<X>>)
                             : (u == 1 ? gated_fp8_kernel<X, 1, 1> : gated_fp8_kernel<X, 1, MANY<X>>);
        launch_overlapped(kernel, dim3(ctas), dim3(ROW_THREADS), 0, stream, (const X*)gate_up, parts, part_stride, (uint8_t*)q, scales, blocks, (unsigned)kblocks, F, g);
    });
    return check_launch("gated_fp8");
}

PH_DEFINE_LAST_ERROR(ph_fp8)
