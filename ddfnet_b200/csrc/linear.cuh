// The matrix products of linear_act on the tensor cores: D (M x N) = A (M x K) B (N x K)^T, 2-byte operands, float
// accumulation, and everything that follows the product on the way out of it.
//
//   forward     y  = act(x W^T + b [+ r]) [+ r]   A = x (K innermost), B = W (K innermost)
//   grad x      gx = gz W                          A = gz (K innermost), B = W with its rows as the reduction
//   grad W      gW = gz^T x                        both operands with their rows as the reduction
// An operand whose reduction axis is not the innermost one needs no transposed copy: the tensor core takes either
// order from shared memory (AT, BT).
//
// What bounds it: 2 M N K operations at the tensor cores' rate, or, with few rows or small K, the operands' and
// results' bytes.  One persistent block an SM:
//   warp 0     one thread loads tiles of 64 along K by TMA into a ring of stages (192 KB)
//   warp 1     one thread issues the products, 128 x BN, into one of two accumulators in tensor memory
//   warps 4-11 take the other accumulator meanwhile: 32 x 32 pieces through shared memory, so that eight
//              lanes read and write 64 bytes of one row
// BN = 256 where the tiles fill the machine: a 128 x 256 tile's operands take 96 bytes of shared memory a clock
// at the full rate, a 128 x 128 tile's all 128.  Smaller BN and splits of K (partial sums in the workspace, joined
// in a fixed order by linear_join_kernel) where they would not.
//
// Every wait is bounded: a role whose wait runs out records a fault and leaves its loop, the others follow by their
// own limits; the block meets after a pause in which its copies land, frees the tensor memory and ends.
#pragma once

#include "tcgen05.cuh"

namespace ddf {

constexpr int kFaultLinear = 6;  // a wait of linear_kernel ran out
constexpr int kTileM = 128, kTileK = 64;
constexpr int kLinearThreads = 384, kJoinWarps = 8;
constexpr uint32_t kRingBytes = 192 * 1024;
constexpr uint32_t kPieceBytes = 32 * 32 * 4;  // an epilogue warp's piece
constexpr uint32_t kLinearShared = kRingBytes + kJoinWarps * kPieceBytes + 1024 + 256;

enum Act { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// The normal distribution's Phi(z), and e = exp(-z^2 / 2).  1 - Phi(a) = exp(-a^2 / 2) g(a) for a >= 0, where g falls
// from 1/2 as 0.4 / a: a polynomial in t = 1 / (1 + 0.315 a) without constant term, fitted for the least relative
// error over [0, 40] (4.0e-7), by iterated weighted least squares.  erff and expf would cost twice the instructions.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float a = fabsf(z), t = __fdividef(1.f, fmaf(0.315f, a, 1.f));
    float g = 0.034466008f;
    g = fmaf(g, t, -0.12912883f);
    g = fmaf(g, t, 0.12538007f);
    g = fmaf(g, t, 0.0050840266f);
    g = fmaf(g, t, 0.10151252f);
    g = fmaf(g, t, 0.1112041f);
    g = fmaf(g, t, 0.1258197f);
    g = fmaf(g, t, 0.12566227f);
    e = exp2_fast(a * a * -0.72134752f);
    const float q = e * (g * t);
    return z > 0.f ? 1.f - q : q;
}
template <int ACT> __device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == kActRelu) return z > 0.f || z != z ? z : 0.f;
    if constexpr (ACT == kActGelu) {
        float e;
        const float phi = normal_cdf(z, e);
        return z != z ? z : z * phi;
    }
    if constexpr (ACT == kActSilu) return __fdividef(z, 1.f + exp2_fast(z * -1.4426950f));
    return z;
}
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == kActRelu) return z > 0.f ? 1.f : (z != z ? z : 0.f);
    if constexpr (ACT == kActGelu) {
        float e;
        const float phi = normal_cdf(z, e);
        return z != z ? z : fmaf(z * 0.39894228f, e, phi);
    }
    if constexpr (ACT == kActSilu) {
        const float s = __fdividef(1.f, 1.f + exp2_fast(z * -1.4426950f));
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}
__device__ __forceinline__ float act_value(float z, int act) {
    return act == kActRelu ? act_value<kActRelu>(z) : act == kActGelu ? act_value<kActGelu>(z) : act == kActSilu ? act_value<kActSilu>(z) : z;
}

// What follows the product.
struct Epilogue {
    void* y;               // M x N, rows ldy apart
    void* aux;             // z = product + bias (+ residual before), or NULL
    const void* bias;      // N, or NULL
    const void* residual;  // rows ldr apart, or NULL
    long long ldy, ldr;
    int act, after;        // after: the residual follows the activation
    int vec;               // y, aux and residual can be accessed by four elements
};

// Four neighbouring elements of a row, the first `n` of them.
template <typename T> __device__ __forceinline__ void load4(const T* p, bool vec, int n, float (&v)[4]) {
    if (vec && n >= 4) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
        v[0] = Word<T>::get(w.x, 0); v[1] = Word<T>::get(w.x, 1);
        v[2] = Word<T>::get(w.y, 0); v[3] = Word<T>::get(w.y, 1);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? Elem<T>::load(p + i) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store4(T* p, bool vec, int n, const float (&v)[4]) {
    if (vec && n >= 4) {
        *reinterpret_cast<uint2*>(p) = make_uint2(Word<T>::put(v[0], v[1]), Word<T>::put(v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) Elem<T>::store(p + i, v[i]);
    }
}

// bias, residual, activation and the stores of four elements of a row: `b` and `r` are 0 where there is none.
template <typename T, int ACT = -1>  // -1: as e.act says
__device__ __forceinline__ void finish4(const Epilogue& e, long long row, int col, int n, float (&z)[4], const float (&b)[4], const float (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        z[i] += b[i];
        if (!e.after) z[i] += r[i];
    }
    if (e.aux) store4(reinterpret_cast<T*>(e.aux) + row * e.ldy + col, e.vec, n, z);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (ACT < 0) z[i] = act_value(z[i], e.act);
        else z[i] = act_value<ACT>(z[i]);
    }
    if (e.after) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] += r[i];
    }
    store4(reinterpret_cast<T*>(e.y) + row * e.ldy + col, e.vec, n, z);
}

struct LinearPlan {
    CUtensorMap a, b;
    Epilogue out;
    float* partial;      // splits x M x N, where splits > 1
    int M, N, K;
    int tiles_m, tiles_n, splits, steps;  // steps of 64 along K in a split
    uint32_t idesc;
    int* fault;
    long long limit;     // of a wait, in clocks
};

// Work item -> tile and split: tiles of eight blocks of rows side by side, so that the tiles in flight share operands.
__device__ __forceinline__ void tile_of(const LinearPlan& p, int item, int& m, int& n, int& split) {
    const int tiles = p.tiles_m * p.tiles_n;
    split = item / tiles;
    const int t = item - split * tiles;
    const int group = t / (8 * p.tiles_n), in = t - group * 8 * p.tiles_n;
    const int rows = min(8, p.tiles_m - group * 8);
    m = group * 8 + in % rows;
    n = in / rows;
}

template <typename T, int BN, bool AT, bool BT, int ACT>
__global__ void __launch_bounds__(kLinearThreads, 1) linear_kernel(const __grid_constant__ LinearPlan p) {
    constexpr uint32_t kA = kTileM * kTileK * 2, kB = BN * kTileK * 2, kStage = kA + kB;
    constexpr int kStages = (int)(kRingBytes / kStage);
    extern __shared__ unsigned char linear_raw[];
    const uint32_t base = (smem_u32(linear_raw) + 1023u) & ~1023u;
    const uint32_t pieces = base + kRingBytes, bars = pieces + kJoinWarps * kPieceBytes;
    const auto full = [&](int s) { return bars + 8u * s; };
    const auto empty = [&](int s) { return bars + 8u * (kStages + s); };
    const auto acc_full = [&](int s) { return bars + 8u * (2 * kStages + s); };
    const auto acc_empty = [&](int s) { return bars + 8u * (2 * kStages + 2 + s); };
    const uint32_t tmem_word = bars + 8u * (2 * kStages + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int items = p.tiles_m * p.tiles_n * p.splits;
    const int all_steps = (p.K + kTileK - 1) / kTileK;
    bool late = false;  // one of this thread's waits ran out

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full(s), 1);
            mbar_init(acc_empty(s), kJoinWarps);
        }
        mbar_fence_init();
        tma_prefetch_map(&p.a);
        tma_prefetch_map(&p.b);
    }
    if (warp == 2) tmem_alloc(tmem_word, 2 * BN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = lds32(tmem_word);

    if (warp == 0 && lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        for (int item = blockIdx.x; item < items && !late; item += gridDim.x) {
            int m, n, split;
            tile_of(p, item, m, n, split);
            const int k1 = min(all_steps, (split + 1) * p.steps);
            for (int k = split * p.steps; k < k1; ++k) {
                if (!mbar_wait_for(empty(stage), phase ^ 1u, p.limit)) { late = true; break; }
                const uint32_t to = base + (uint32_t)stage * kStage;
                mbar_arrive_expect_tx(full(stage), kStage);
                if constexpr (AT) {
#pragma unroll
                    for (int i = 0; i < kTileM / 64; ++i)
                        tma_load_2d(to + i * 64 * kTileK * 2, &p.a, m * kTileM + i * 64, k * kTileK, full(stage));
                } else {
                    tma_load_2d(to, &p.a, k * kTileK, m * kTileM, full(stage));
                }
                if constexpr (BT) {
#pragma unroll
                    for (int i = 0; i < BN / 64; ++i)
                        tma_load_2d(to + kA + i * 64 * kTileK * 2, &p.b, n * BN + i * 64, k * kTileK, full(stage));
                } else {
                    tma_load_2d(to + kA, &p.b, k * kTileK, n * BN, full(stage));
                }
                if (++stage == kStages) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1 && lane == 0) {
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        for (int item = blockIdx.x; item < items && !late; item += gridDim.x) {
            int m, n, split;
            tile_of(p, item, m, n, split);
            if (!mbar_wait_for(acc_empty(acc), acc_phase ^ 1u, p.limit)) { late = true; break; }
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(acc * BN);
            const int k0 = split * p.steps, k1 = min(all_steps, k0 + p.steps);
            for (int k = k0; k < k1; ++k) {
                if (!mbar_wait_for(full(stage), phase, p.limit)) { late = true; break; }
                tc_fence_after();
                const uint32_t from = base + (uint32_t)stage * kStage;
#pragma unroll
                for (int j = 0; j < kTileK / 16; ++j) {
                    // 16 along K: 32 bytes of every row, or 16 rows
                    const uint64_t da = smem_descriptor(from + (AT ? j * 2048 : j * 32), AT ? 64 * kTileK * 2 : 16);
                    const uint64_t db = smem_descriptor(from + kA + (BT ? j * 2048 : j * 32), BT ? 64 * kTileK * 2 : 16);
                    tc_mma(d, da, db, p.idesc, k > k0 || j > 0);
                }
                tc_commit(empty(stage));
                if (++stage == kStages) { stage = 0; phase ^= 1u; }
            }
            tc_commit(acc_full(acc));
            if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t piece = pieces + (uint32_t)(warp - 4) * kPieceBytes;
        const int sub = lane & 7;  // four columns of a piece
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int item = blockIdx.x; item < items; item += gridDim.x) {
            int m, n, split;
            tile_of(p, item, m, n, split);
            if (!mbar_wait_for(acc_full(acc), acc_phase, p.limit)) { late = true; break; }
            tc_fence_after();
            const int row0 = m * kTileM + quarter * 32 + (lane >> 3);
            const bool whole = m * kTileM + kTileM <= p.M && n * BN + BN <= p.N && (p.partial ? (p.N & 3) == 0 : p.out.vec != 0);
#pragma unroll 1
            for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
                const int col = n * BN + c + sub * 4;
                uint2 rw[8];
                float b[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t v[32];
                tmem_load32(tmem + (uint32_t)(acc * BN + c) + ((uint32_t)quarter << 21), v);
                if (whole && !p.partial) {  // on their way while the accumulator is read
                    if (p.out.residual) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            rw[i] = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(p.out.residual) + (long long)(row0 + i * 4) * p.out.ldr + col));
                    }
                    if (p.out.bias) load4(reinterpret_cast<const T*>(p.out.bias) + col, false, 4, b);
                }
                tmem_wait_load();
                if (c + 32 >= (half + 1) * (BN / 2)) {  // the accumulator's last piece is in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty(acc));
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece + lane * 128 + ((i ^ (lane & 7)) * 16)),
                                 "r"(v[4 * i]), "r"(v[4 * i + 1]), "r"(v[4 * i + 2]), "r"(v[4 * i + 3])
                                 : "memory");
                __syncwarp();
                if (whole) {
                    float z[8][4];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int in = i * 4 + (lane >> 3);
                        uint32_t w[4];
                        lds128(piece + in * 128 + ((sub ^ (in & 7)) * 16), w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[i][j] = __uint_as_float(w[j]) + b[j];
                    }
                    if (p.partial) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<float4*>(p.partial + ((long long)split * p.M + row0 + i * 4) * p.N + col) =
                                make_float4(z[i][0], z[i][1], z[i][2], z[i][3]);
                    } else {
                        const auto residual = [&] {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                z[i][0] += Word<T>::get(rw[i].x, 0);
                                z[i][1] += Word<T>::get(rw[i].x, 1);
                                z[i][2] += Word<T>::get(rw[i].y, 0);
                                z[i][3] += Word<T>::get(rw[i].y, 1);
                            }
                        };
                        const auto store = [&](void* to) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<uint2*>(reinterpret_cast<T*>(to) + (long long)(row0 + i * 4) * p.out.ldy + col) =
                                    make_uint2(Word<T>::put(z[i][0], z[i][1]), Word<T>::put(z[i][2], z[i][3]));
                        };
                        if (p.out.residual && !p.out.after) residual();
                        if (p.out.aux) store(p.out.aux);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) z[i][j] = act_value<ACT>(z[i][j]);
                        if (p.out.residual && p.out.after) residual();
                        store(p.out.y);
                    }
                } else {
                    const int left = p.N - col;
                    if (!p.partial && p.out.bias && left > 0) load4(reinterpret_cast<const T*>(p.out.bias) + col, false, left, b);
#pragma unroll 1
                    for (int i = 0; i < 8; ++i) {
                        const int in = i * 4 + (lane >> 3);
                        const long long row = row0 + i * 4;
                        uint32_t w[4];
                        lds128(piece + in * 128 + ((sub ^ (in & 7)) * 16), w[0], w[1], w[2], w[3]);
                        if (row >= p.M || left <= 0) continue;
                        float z[4] = {__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3])};
                        if (p.partial) {
                            float* to = p.partial + ((long long)split * p.M + row) * p.N + col;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (j < left) to[j] = z[j];
                        } else {
                            float r[4] = {0.f, 0.f, 0.f, 0.f};
                            if (p.out.residual) load4(reinterpret_cast<const T*>(p.out.residual) + row * p.out.ldr + col, p.out.vec, left, r);
                            finish4<T, ACT>(p.out, row, col, left, z, b, r);
                        }
                    }
                }
                __syncwarp();
            }
            if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
    }
    if (late) {
        atomicCAS(p.fault, 0, kFaultLinear);
        // what is in flight (copies, products) ends in microseconds
        for (int i = 0; i < 100; ++i) __nanosleep(100000);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 2) tmem_free(tmem, 2 * BN);
}

// Joins the splits of K in their order and finishes: four elements a thread.
template <typename T> __global__ void __launch_bounds__(256) linear_join_kernel(const float* __restrict__ partial, const Epilogue out, int M, int N, int splits) {
    const int quads = (N + 3) / 4;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = at / quads;
    if (row >= M) return;
    const int col = (int)(at - row * quads) * 4, left = N - col;
    float z[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
    const bool vec = (N & 3) == 0;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float* from = partial + ((long long)s * M + row) * N + col;
        if (vec) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(from));
            z[0] += v.x; z[1] += v.y; z[2] += v.z; z[3] += v.w;
        } else {
            for (int j = 0; j < 4; ++j)
                if (j < left) z[j] += __ldg(from + j);
        }
    }
    if (out.bias) load4(reinterpret_cast<const T*>(out.bias) + col, false, left, b);
    if (out.residual) load4(reinterpret_cast<const T*>(out.residual) + row * out.ldr + col, out.vec, left, r);
    finish4<T>(out, row, col, left, z, b, r);
}

}  // namespace ddf
