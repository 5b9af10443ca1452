// 8-bit projections: y[i][j] = sx[i] sw[j] sum_k q[i][k] W[j][k] (+ bias[j]), q and W in int8, the sum exact in int32.
//
// Quantised rows.  With a = max_k |x_k|:  scale = a / 127 (rounded to FP32),  q_k = 127 x_k / a rounded to the nearest whole
// number, ties to even, of the exact quotient, so that the integers do not depend on the order of two roundings.  A row of
// zeros has scale 0; a row that holds an infinity or a NaN gets zeros and the scale NaN, so all its products are NaN.
#pragma once
#include <cuda_bf16.h>
#include <type_traits>

#include "sd_common.cuh"
#include "sd_tc.cuh"

namespace sd {

// ---- quantised rows -----------------------------------------------------------------------------------------------
struct QuantizeParams {
    long long rows;
    int K;
    const void* x;
    long long x_stride;   // elements
    signed char* q;
    long long q_stride;   // bytes
    float* scale;
};

// What a row's largest magnitude (its bits) makes of the row.
struct RowScale {
    float scale, inverse, largest;   // a / 127, about 127 / a, a
    bool bad, special;               // not finite; that, or at either end of FP32's range: see quantize_extreme
};
__device__ __forceinline__ RowScale row_scale(unsigned largest_bits) {
    RowScale r;
    r.largest = __uint_as_float(largest_bits);
    r.bad = largest_bits >= 0x7f800000u;
    r.special = r.largest < 1e-30f || !(r.largest < 2.5e36f);
    r.scale = r.bad ? __uint_as_float(0x7fffffffu) : __fdiv_rn(r.largest, 127.f);
    r.inverse = r.special ? 0.f : __fdiv_rn(127.f, r.largest);
    return r;
}
// 127 x / a rounded to nearest even.  The product with the rounded inverse is less than a half off, so the quotient lies between
// the neighbours of the half h above its whole part; 127 x and h a, each with what FP32 rounds off, are compared exactly.  (BF16
// rows come here often: the half of their largest entry is a tie.)
__device__ __forceinline__ int quantize_exactly(float x, float inverse, float a) {
    const float low = floorf(x * inverse), h = low + 0.5f, l = 127.f * x, r = h * a;
    const float dl = fmaf(127.f, x, -l), dr = fmaf(h, a, -r);
    const bool above = l > r || (l == r && dl > dr), tie = l == r && dl == dr;
    const int n = (int)low;
    return n + (above || (tie && (n & 1)) ? 1 : 0);
}
// The same for rows whose inverse, or whose 127 x, may overflow.  (A quotient that is not a half is 2^-40 of itself or more off one.)
__device__ __noinline__ int quantize_extreme(float x, float a) { return a == 0.f ? 0 : (int)rint(127.0 * (double)x / (double)a); }

template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Eight entries of a row as they lie in memory.
template <class T>
struct Piece {
    uint4 raw[sizeof(T) / 2];
};
// From column c0 on, zeros past the row's end.  VEC: rows start on 16-byte boundaries and K is a multiple of eight, so that a
// request is one predicated instruction and a lane's requests go out together.
template <class T, bool VEC>
__device__ __forceinline__ Piece<T> load_piece(const T* row, int c0, int K) {
    Piece<T> p;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) p.raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
            if (c0 < K) p.raw[i] = reinterpret_cast<const uint4*>(row + c0)[i];
    } else {
        T* e = reinterpret_cast<T*>(p.raw);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < K) e[i] = row[c0 + i];
    }
    return p;
}
// The larger of `top` and the entries' magnitudes, as FP32 bits but not yet reduced: piece_top() of BF16 keeps the even and the
// odd entries' bits in two halves (infinities and NaNs are the largest numbers there as well).
template <class T>
__device__ __forceinline__ unsigned piece_top(const Piece<T>& p, unsigned top) {
    const unsigned* w = reinterpret_cast<const unsigned*>(p.raw);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 2; ++i)
        top = sizeof(T) == 2 ? __vmaxu2(top, w[i] & 0x7fff7fffu) : max(top, w[i] & 0x7fffffffu);
    return top;
}
template <class T>
__device__ __forceinline__ unsigned whole_top(unsigned top) { return sizeof(T) == 2 ? max(top & 0xffff0000u, top << 16) : top; }

// The entries as bytes.  With b = 384.5 + 2^-15 the sum 127 x / a + b has eight bits of q + 128 and 15 bits behind the point; the
// product with the inverse, which is rounded to 2^-24 of itself, and the sum are off by less than 2^-15 together (2^-17, and half a
// unit: 2^-16), so q is right unless those 15 bits are 0, 1 or 2, next to where it changes.
template <class T>
__device__ __forceinline__ uint2 quantize_piece(const Piece<T>& p, const RowScale& r) {
    float v[8];
    unsigned u[8], near = 0xffffffffu;
    if constexpr (sizeof(T) == 2) {
        const unsigned* w = reinterpret_cast<const unsigned*>(p.raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const float* f = reinterpret_cast<const float*>(p.raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = f[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        u[i] = __float_as_uint(fmaf(v[i], r.inverse, 384.5f + 0x1p-15f));
        near = min(near, u[i] & 0x7fffu);
        u[i] <<= 1;   // q + 128 in the third byte
    }
    if (near <= 2 || r.special) {
        if (!r.special) {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = (unsigned)(quantize_exactly(v[i], r.inverse, r.largest) + 128) << 16;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = (unsigned)((r.bad ? 0 : quantize_extreme(v[i], r.largest)) + 128) << 16;
        }
    }
    uint2 out;
    out.x = __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410) ^ 0x80808080u;
    out.y = __byte_perm(__byte_perm(u[4], u[5], 0x0062), __byte_perm(u[6], u[7], 0x0062), 0x5410) ^ 0x80808080u;
    return out;
}

// Groups of W warps take a row each, eight rows to W = 1 in a CTA; a lane keeps up to H pieces of eight entries between the
// search for the largest magnitude and the rounding (longer rows are read again).  q rows start on 16-byte boundaries,
// q_stride covers K rounded up to 16, and the bytes past K are set to zero.
constexpr int QUANT_THREADS = 256;
template <class T, bool VEC, int W, int H>
__global__ void __launch_bounds__(QUANT_THREADS) k_quantize_rows(QuantizeParams p) {
    __shared__ unsigned s_max[QUANT_THREADS / 32];
    chain_wait();
    chain_release();
    const int warp = threadIdx.x >> 5, at = (warp % W) * 32 + (threadIdx.x & 31);
    const long long r_idx = (long long)blockIdx.x * (8 / W) + warp / W;
    const bool live = r_idx < p.rows;   // the rows of a CTA share its barrier
    const T* row = reinterpret_cast<const T*>(p.x) + (live ? r_idx : 0) * p.x_stride;
    Piece<T> held[H];
    unsigned top = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) held[h] = load_piece<T, VEC>(row, (h * W * 32 + at) * 8, p.K);
#pragma unroll
    for (int h = 0; h < H; ++h) top = piece_top(held[h], top);
    for (int c0 = (H * W * 32 + at) * 8; c0 < p.K; c0 += W * 256) top = piece_top(load_piece<T, VEC>(row, c0, p.K), top);
    top = whole_top<T>(top);
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (W > 1) {
        if ((threadIdx.x & 31) == 0) s_max[warp] = top;
        __syncthreads();
        top = __reduce_max_sync(0xffffffffu, s_max[warp / W * W + threadIdx.x % W]);
    }
    if (!live) return;
    const RowScale r = row_scale(top);
    signed char* out = p.q + r_idx * p.q_stride;
    const int padded = (p.K + 15) / 16 * 16;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const int c0 = (h * W * 32 + at) * 8;
        if (c0 < padded) *reinterpret_cast<uint2*>(out + c0) = quantize_piece(held[h], r);
    }
    for (int c0 = (H * W * 32 + at) * 8; c0 < padded; c0 += W * 256)
        *reinterpret_cast<uint2*>(out + c0) = quantize_piece(load_piece<T, VEC>(row, c0, p.K), r);
    if (at == 0) p.scale[r_idx] = r.scale;
}

// ---- the product --------------------------------------------------------------------------------------------------
struct Int8Params {
    int M, outs, K;            // rows, output columns (half of the weight's rows with SwiGLU), length of the sums
    const float* x_scale;      // [M]
    const float* w_scale;      // [N]
    const void* bias;          // [N] or null
    int bias_f32;
    void* y;
    long long y_stride;        // elements
    int out_f32;
    int tiles_m, tiles_n;
};

__device__ __forceinline__ float int8_bias(const Int8Params& p, int n) {
    if (p.bias == nullptr) return 0.f;
    return p.bias_f32 ? reinterpret_cast<const float*>(p.bias)[n]
                      : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias)[n]);
}
// silu(gate) * value, both in FP32, rounded once by the store
__device__ __forceinline__ float int8_gated(float gate, float value) { return gate * sigmoidf_(gate) * value; }

// tcgen05.mma.kind::i8, int32 accumulators in tensor memory, both operands K-major in shared memory as rows of 128 bytes with
// the 128-byte swizzle, loaded by TMA (which fills what lies outside with zeros: ragged M, N and K need nothing else) into a
// ring of stages.  Persistent: one thread loads, one issues the products, eight warps empty the accumulator, of which there
// are two, so that the products of a tile run under the epilogue of the one before.  With SwiGLU half of a tile's weight rows
// are gate rows and half the value rows that belong to them, so that its accumulator holds both factors of its outputs.
//
// PAIR: two CTAs of a cluster share a tile of 256 rows by 256 weight rows (cta_group::2): each loads 128 of either, the first
// one's thread issues for both, each holds 128 rows of the accumulator.  One CTA by itself with 128 x 256 moves 12 KB of
// operands for an instruction of 128 clocks and receives as much, more than the 128 bytes a clock of its shared memory; a pair
// moves 8 KB.  Without PAIR tiles are 128 rows by BN, for few rows or few tiles.
constexpr int I8_BM = 128, I8_BK = 128, I8_THREADS = 384, I8_EPILOGUE_WARP = 4, I8_EPILOGUE_THREADS = 256;
constexpr int I8_GROUP = 8;   // row tiles that are walked together: their rows and the weight tiles stay in L2
constexpr int I8_STAGING = 32 * 64;   // bytes of a warp, see int8_store
template <int BN, bool PAIR>
struct Int8Tile {
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;   // weight rows that a CTA loads
    static constexpr unsigned A_BYTES = I8_BM * I8_BK, B_BYTES = B_ROWS * I8_BK, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = 192 * 1024 / STAGE_BYTES;
    static constexpr unsigned TMEM_COLS = 2 * BN;
    static constexpr size_t SMEM = size_t(STAGES) * STAGE_BYTES + 8 * I8_STAGING + 1024;
};

template <bool PAIR>
__device__ __forceinline__ void i8_load(unsigned smem, const CUtensorMap* map, int col, int row, unsigned bar) {
    if constexpr (PAIR)   // the barrier may be the other CTA's
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem),
            "l"(reinterpret_cast<unsigned long long>(map)), "r"(col), "r"(row), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem),
            "l"(reinterpret_cast<unsigned long long>(map)), "r"(col), "r"(row), "r"(bar)
            : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void i8_mma(unsigned d_tmem, unsigned long long da, unsigned long long db, unsigned idesc,
                                       unsigned accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives on `bar` when all products issued so far are done; with PAIR on the barriers at that place in both CTAs.
template <bool PAIR>
__device__ __forceinline__ void i8_commit(unsigned bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((unsigned short)3)
                     : "memory");
    else
        tc_commit(bar);
}
// int32 accumulator (2 at bit 4), signed operands (1 at bits 7 and 10), both K-major
__host__ __device__ constexpr unsigned i8_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
}

// 64 bytes of each of a warp's 32 rows, a lane's row in v, from output column `col` on.  Stored as they lie in the lanes a
// request would touch 32 rows with half a sector each; through shared memory (16-byte pieces, exchanged by row so that eight
// lanes use all banks) four lanes store a row's 64 bytes.
template <bool F32>
__device__ __forceinline__ void int8_store(const Int8Params& p, unsigned char* staging, int row0, int col, const float* v, bool vec) {
    constexpr int PER = F32 ? 4 : 8, COLS = 4 * PER;
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint4 w;
        if constexpr (F32) {
            w = make_uint4(__float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]), __float_as_uint(v[4 * c + 2]), __float_as_uint(v[4 * c + 3]));
        } else {
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[8 * c + 2 * e], v[8 * c + 2 * e + 1]);
        }
        *reinterpret_cast<uint4*>(staging + lane * 64 + ((c ^ (lane >> 1)) & 3) * 16) = w;
    }
    __syncwarp();
    using Out = typename std::conditional<F32, float, __nv_bfloat16>::type;
    Out* y = reinterpret_cast<Out*>(p.y);
    if (vec && col + COLS <= p.outs) {
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int r = it * 8 + (lane >> 2), c = lane & 3;
            const uint4 w = *reinterpret_cast<const uint4*>(staging + r * 64 + ((c ^ (r >> 1)) & 3) * 16);
            if (row0 + r < p.M) *reinterpret_cast<uint4*>(y + (row0 + r) * p.y_stride + col + c * PER) = w;
        }
        return;
    }
    // rows that start anywhere, or the last columns: an entry a lane
    for (int idx = lane; idx < 32 * COLS; idx += 32) {
        const int r = idx / COLS, e = idx % COLS;
        if (row0 + r < p.M && col + e < p.outs)
            y[(row0 + r) * p.y_stride + col + e] =
                reinterpret_cast<const Out*>(staging + r * 64 + (((e / PER) ^ (r >> 1)) & 3) * 16)[e % PER];
    }
}

// The scales and biases of a tile's weight rows, by the epilogue's threads (OUTS output columns from column0 on; with GATED the
// value rows' behind them).
template <int BN, bool GATED>
__device__ __forceinline__ void int8_columns(const Int8Params& p, int column0, float* scale, float* bias) {
    constexpr int OUTS = GATED ? BN / 2 : BN;
    const int i = threadIdx.x - I8_EPILOGUE_WARP * 32;
    if (i >= BN) return;
    const int col = column0 + (GATED ? i % OUTS : i), w = GATED && i >= OUTS ? p.outs + col : col;
    scale[i] = col < p.outs ? p.w_scale[w] : 0.f;
    bias[i] = col < p.outs ? int8_bias(p, w) : 0.f;
}
// A row's sums v (and g, of the value rows) of STEP columns from c0 of the tile on -> outputs in v.
template <int STEP, bool GATED>
__device__ __forceinline__ void int8_finish(const Int8Params& p, float (&v)[STEP], float (&g)[GATED ? STEP : 1], float sx, const float* scale,
                                            const float* bias, int c0, int values) {
    // (shared memory is what the products are short of: without a bias none is read)
#pragma unroll
    for (int e = 0; e < STEP; ++e) {
        v[e] = (float)__float_as_int(v[e]) * sx * scale[c0 + e];
        if constexpr (GATED) g[e] = (float)__float_as_int(g[e]) * sx * scale[values + c0 + e];
    }
    if (p.bias != nullptr) {
#pragma unroll
        for (int e = 0; e < STEP; ++e) {
            v[e] += bias[c0 + e];
            if constexpr (GATED) g[e] += bias[values + c0 + e];
        }
    }
    if constexpr (GATED) {
#pragma unroll
        for (int e = 0; e < STEP; ++e) v[e] = int8_gated(v[e], g[e]);
    }
}

template <int BN, bool GATED, bool F32, bool PAIR>
__global__ void __launch_bounds__(I8_THREADS, 1)
k_int8_matmul(Int8Params p, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, int* fault) {
    using Tile = Int8Tile<BN, PAIR>;
    constexpr int S = Tile::STAGES, OUTS = GATED ? BN / 2 : BN, BM = PAIR ? 2 * I8_BM : I8_BM, CTAS = PAIR ? 2 : 1;
    extern __shared__ __align__(16) unsigned char i8_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * S + 4];   // full, empty, accumulator full, accumulator empty
    __shared__ unsigned s_tmem;
    __shared__ __align__(16) float s_scale[2][BN], s_bias[2][BN];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = PAIR ? blockIdx.x & 1 : 0;
    const unsigned ring = (tc_smem(i8_raw) + 1023u) & ~1023u;
    unsigned char* const staging = i8_raw + (ring - tc_smem(i8_raw)) + S * Tile::STAGE_BYTES + (warp & 7) * I8_STAGING;
    const unsigned full0 = tc_smem(bars), empty0 = full0 + 8 * S, acc_full0 = empty0 + 8 * S, acc_empty0 = acc_full0 + 16;
    const auto pair_barrier = [&]() {
        if constexpr (PAIR) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
        else __syncthreads();
    };

    if (tid == 0) {
        for (int i = 0; i < 2 * S + 2; ++i)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full0 + 8 * i));
        for (int i = 0; i < 2; ++i)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(acc_empty0 + 8 * i), "r"(CTAS * I8_EPILOGUE_THREADS));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&s_tmem)), "r"(Tile::TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&s_tmem)), "r"(Tile::TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        }
    }
    if (warp == 3 && lane < 2)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<unsigned long long>(lane == 0 ? &x_map : &w_map)) : "memory");
    tc_fence_before();
    pair_barrier();
    tc_fence_after();
    chain_wait();   // the set-up above runs under the kernel that writes the rows
    chain_release();
    const unsigned tbase = s_tmem;
    const int tiles = p.tiles_m * p.tiles_n, blocks = (p.K + I8_BK - 1) / I8_BK;
    const int worker = blockIdx.x / CTAS, workers = gridDim.x / CTAS;
    // groups of I8_GROUP row tiles; inside one, the row tile changes first
    const auto place = [&](int tile, int& m, int& n) {
        const int per_group = I8_GROUP * p.tiles_n, g = tile / per_group, rest = tile - g * per_group;
        const int height = min(I8_GROUP, p.tiles_m - g * I8_GROUP);
        n = rest / height;
        m = g * I8_GROUP + rest - n * height;
    };
    // a barrier of the pair's first CTA
    const auto of_first = [&](unsigned bar) {
        unsigned a = bar;
        if constexpr (PAIR) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(bar));
        return a;
    };

    if (warp == 0) {   // ---- loads
        if (lane == 0) {
            int k = 0;   // stages filled so far
            bool alive = true;
            for (int tile = worker; tile < tiles && alive; tile += workers) {
                int m, n;
                place(tile, m, n);
                for (int b = 0; b < blocks; ++b, ++k) {
                    const int s = k % S;
                    if (k >= S) alive = tc_wait(empty0 + 8 * s, (k / S - 1) & 1);
                    if (!alive) break;
                    const unsigned bar = of_first(full0 + 8 * s), a = ring + s * Tile::STAGE_BYTES, w = a + Tile::A_BYTES;
                    if (rank == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full0 + 8 * s),
                                     "r"(CTAS * Tile::STAGE_BYTES)
                                     : "memory");
                    i8_load<PAIR>(a, &x_map, b * I8_BK, m * BM + rank * I8_BM, bar);
                    if constexpr (PAIR) {   // the gate rows or the value rows; or either half
                        i8_load<PAIR>(w, &w_map, b * I8_BK, GATED ? rank * p.outs + n * OUTS : n * OUTS + rank * Tile::B_ROWS, bar);
                    } else {
                        i8_load<PAIR>(w, &w_map, b * I8_BK, n * OUTS, bar);
                        if (GATED) i8_load<PAIR>(w + Tile::B_BYTES / 2, &w_map, b * I8_BK, p.outs + n * OUTS, bar);
                    }
                }
            }
            // with PAIR the first CTA's arrivals reach this one's memory: none is on its way when it leaves
            for (int i = k > S ? k - S : 0; PAIR && i < k && alive; ++i) alive = tc_wait(empty0 + 8 * (i % S), (i / S) & 1);
            if (!alive) {
                atomicExch(fault, 9);
                // copies in flight, into this CTA and (PAIR) the other, land before anyone leaves
                if (rank == 0)
                    for (int i = k > S ? k - S : 0; i < k; ++i) tc_wait(full0 + 8 * (i % S), (i / S) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {   // ---- products
        if (lane == 0 && rank == 0) {
            int k = 0, t = 0;
            bool alive = true;
            for (int tile = worker; tile < tiles && alive; tile += workers, ++t) {
                if (t >= 2) alive = tc_wait(acc_empty0 + 8 * (t & 1), (t / 2 - 1) & 1);
                tc_fence_after();
                const unsigned acc = tbase + (t & 1) * BN;
                for (int b = 0; b < blocks && alive; ++b, ++k) {
                    const int s = k % S;
                    alive = tc_wait(full0 + 8 * s, (k / S) & 1);
                    if (!alive) break;
                    tc_fence_after();
                    const unsigned a = ring + s * Tile::STAGE_BYTES, w = a + Tile::A_BYTES;
#pragma unroll
                    for (int j = 0; j < I8_BK / 32; ++j)
                        i8_mma<PAIR>(acc, tc_desc(a + j * 32, 16, 1024) | (2ull << 61), tc_desc(w + j * 32, 16, 1024) | (2ull << 61),
                                     i8_idesc(BM, BN), b > 0 || j > 0 ? 1u : 0u);
                    i8_commit<PAIR>(empty0 + 8 * s);
                }
                if (alive) i8_commit<PAIR>(acc_full0 + 8 * (t & 1));
            }
            if (!alive) atomicExch(fault, 10);
        }
        __syncwarp();
    } else if (warp >= I8_EPILOGUE_WARP) {   // ---- scales, bias, gate, store
        const int quarter = warp & 3, half = (warp - I8_EPILOGUE_WARP) >> 2;
        const bool vec = (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && p.y_stride % (F32 ? 4 : 8) == 0;
        int t = 0;
        bool alive = true;
        for (int tile = worker; tile < tiles; tile += workers, ++t) {
            int m, n;
            place(tile, m, n);
            float *scale = s_scale[t & 1], *bias = s_bias[t & 1];
            int8_columns<BN, GATED>(p, n * OUTS, scale, bias);
            asm volatile("bar.sync 1, %0;" ::"n"(I8_EPILOGUE_THREADS) : "memory");
            const int row0 = m * BM + rank * I8_BM + quarter * 32;
            const float sx = row0 + lane < p.M ? p.x_scale[row0 + lane] : 0.f;
            if (alive) alive = tc_wait(acc_full0 + 8 * (t & 1), (t / 2) & 1);
            alive = __all_sync(0xffffffffu, alive);
            if (!alive) {
                if (lane == 0) atomicExch(fault, 11);
                continue;   // nothing is read or stored any more
            }
            tc_fence_after();
            const unsigned acc = tbase + (t & 1) * BN + ((unsigned)(quarter * 32) << 16);
            constexpr int STEP = F32 ? 16 : 32;   // 64 bytes of a row
#pragma unroll 1
            for (int c0 = half * STEP; c0 < OUTS; c0 += 2 * STEP) {
                if (row0 >= p.M || n * OUTS + c0 >= p.outs) break;
                float v[STEP], g[GATED ? STEP : 1];
                tc_ld<STEP>(acc + c0, v);
                if constexpr (GATED) tc_ld<STEP>(acc + OUTS + c0, g);
                tc_wait_ld();
                int8_finish<STEP, GATED>(p, v, g, sx, scale, bias, c0, OUTS);
                int8_store<F32>(p, staging, row0, n * OUTS + c0, v, vec);
            }
            tc_fence_before();
            const unsigned bar = of_first(acc_empty0 + 8 * (t & 1));
            asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
        }
    }
    tc_fence_before();
    pair_barrier();   // with PAIR: nobody leaves while the other may arrive here, load here or read its operands here
    if (warp == 2) {
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(Tile::TMEM_COLS));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(Tile::TMEM_COLS));
    }
}

// The same product where tiles of 128 x 64 are too few for the SMs and the sums are long: the 2, 4 or 8 CTAs of a cluster take
// a tile together, a part of K each (one SM receives some 40 bytes a clock, so that K = 5632 takes it 14 us alone).  Then each
// gets every CTA's sums of its own 64 / CTAS columns, in its ring, which is free by then, adds them up, exactly, and stores.
constexpr int I8_SPLIT_BN = 64;

template <bool GATED, bool F32>
__global__ void __launch_bounds__(I8_THREADS, 1)
k_int8_split(Int8Params p, int ctas_log2, int per, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, int* fault) {
    using Tile = Int8Tile<I8_SPLIT_BN, false>;
    constexpr int S = Tile::STAGES, BN = I8_SPLIT_BN, OUTS = GATED ? BN / 2 : BN;
    extern __shared__ __align__(16) unsigned char i8_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * S + 1];   // full, empty, accumulator full
    __shared__ unsigned s_tmem;
    __shared__ __align__(16) float s_scale[BN], s_bias[BN];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ctas = 1 << ctas_log2, rank = blockIdx.x & (ctas - 1),
              tile = blockIdx.x >> ctas_log2;
    const unsigned ring = (tc_smem(i8_raw) + 1023u) & ~1023u;
    unsigned char* const parts = i8_raw + (ring - tc_smem(i8_raw));
    const unsigned full0 = tc_smem(bars), empty0 = full0 + 8 * S, acc_full = empty0 + 8 * S;
    const auto everywhere = [] { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); };

    if (tid == 0) {
        for (int i = 0; i < 2 * S + 1; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full0 + 8 * i));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&s_tmem)), "r"(BN));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (warp == 3 && lane < 2)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<unsigned long long>(lane == 0 ? &x_map : &w_map)) : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    chain_wait();
    chain_release();
    const unsigned tbase = s_tmem;
    const int m = tile % p.tiles_m, n = tile / p.tiles_m;
    const int blocks = (p.K + I8_BK - 1) / I8_BK, first = rank * per, count = min(per, blocks - first);   // none: nothing is added
    const int quarter = warp & 3, half = (warp - I8_EPILOGUE_WARP) >> 2, row0 = m * I8_BM + quarter * 32;
    const bool epilogue = warp >= I8_EPILOGUE_WARP;
    bool alive = true;

    if (warp == 0 && lane == 0) {
        int k = 0;
        for (; k < count; ++k) {
            const int s = k % S;
            if (k >= S) alive = tc_wait(empty0 + 8 * s, (k / S - 1) & 1);
            if (!alive) break;
            const unsigned bar = full0 + 8 * s, a = ring + s * Tile::STAGE_BYTES, w = a + Tile::A_BYTES;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(Tile::STAGE_BYTES) : "memory");
            i8_load<false>(a, &x_map, (first + k) * I8_BK, m * I8_BM, bar);
            i8_load<false>(w, &w_map, (first + k) * I8_BK, n * OUTS, bar);
            if (GATED) i8_load<false>(w + Tile::B_BYTES / 2, &w_map, (first + k) * I8_BK, p.outs + n * OUTS, bar);
        }
        if (!alive) {
            atomicExch(fault, 9);
            for (int i = k > S ? k - S : 0; i < k; ++i) tc_wait(full0 + 8 * (i % S), (i / S) & 1);   // copies in flight
        }
    } else if (warp == 1 && lane == 0) {
        for (int k = 0; k < count && alive; ++k) {
            const int s = k % S;
            alive = tc_wait(full0 + 8 * s, (k / S) & 1);
            if (!alive) break;
            tc_fence_after();
            const unsigned a = ring + s * Tile::STAGE_BYTES, w = a + Tile::A_BYTES;
#pragma unroll
            for (int j = 0; j < I8_BK / 32; ++j)
                i8_mma<false>(tbase, tc_desc(a + j * 32, 16, 1024) | (2ull << 61), tc_desc(w + j * 32, 16, 1024) | (2ull << 61),
                              i8_idesc(I8_BM, BN), k > 0 || j > 0 ? 1u : 0u);
            i8_commit<false>(empty0 + 8 * s);
        }
        if (alive && count > 0) i8_commit<false>(acc_full);
        if (!alive) atomicExch(fault, 10);
    } else if (epilogue) {
        int8_columns<BN, GATED>(p, n * OUTS, s_scale, s_bias);
        alive = count <= 0 || tc_wait(acc_full, 0);
        alive = __all_sync(0xffffffffu, alive);
        if (!alive && lane == 0) atomicExch(fault, 11);
        tc_fence_after();
    }
    __syncwarp();
    everywhere();   // all products are done: the rings are free
    // A CTA's part: from every CTA `width` columns of 128 rows; with GATED half of them gate and half value columns.
    const int width_log2 = 6 - ctas_log2, width = 1 << width_log2, half_log2 = width_log2 - (GATED ? 1 : 0);
    if (epilogue && alive && count > 0 && row0 < p.M) {
        float v[32];
        tc_ld32(tbase + ((unsigned)(quarter * 32) << 16) + half * 32, v);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const int col = half * 32 + e, in = GATED ? e : col;   // column of the tile, and among the gates (values)
            const int to = in >> half_log2, local = (in & ((1 << half_log2) - 1)) + (GATED && half == 1 ? width / 2 : 0);
            unsigned at;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                         : "=r"(at)
                         : "r"(ring + (((rank << width_log2) + local) * I8_BM + quarter * 32 + lane) * 4), "r"(to));
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "f"(v[e]) : "memory");
        }
    }
    everywhere();
    const int outs = GATED ? width / 2 : width, col0 = rank * outs;   // of the tile
    if (epilogue && alive && row0 + lane < p.M) {
        const int row = row0 + lane;
        const float sx = p.x_scale[row];
        const int* part = reinterpret_cast<const int*>(parts) + quarter * 32 + lane;
        const int active = (blocks + per - 1) / per;
        const auto sum = [&](int local) {
            int v = 0;
            for (int r = 0; r < active; ++r) v += part[((r << width_log2) + local) * I8_BM];
            return (float)v * sx;
        };
        constexpr int STEP = 2;   // neighbouring columns, one store where rows allow it
        const bool vec = (reinterpret_cast<uintptr_t>(p.y) & 7) == 0 && p.y_stride % STEP == 0;
        for (int c = half * STEP; c < outs; c += 2 * STEP) {
            float v[STEP];
#pragma unroll
            for (int e = 0; e < STEP; ++e) {
                const int i = col0 + c + e;
                v[e] = sum(c + e) * s_scale[i] + s_bias[i];
                if constexpr (GATED) v[e] = int8_gated(v[e], sum(outs + c + e) * s_scale[OUTS + i] + s_bias[OUTS + i]);
            }
            const int col = n * OUTS + col0 + c;
            const long long at = row * p.y_stride + col;
            if constexpr (F32) {
                float* y = reinterpret_cast<float*>(p.y) + at;
                if (vec && col + STEP <= p.outs) *reinterpret_cast<float2*>(y) = make_float2(v[0], v[1]);
                else
                    for (int e = 0; e < STEP && col + e < p.outs; ++e) y[e] = v[e];
            } else {
                __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(p.y) + at;
                if (vec && col + STEP <= p.outs) *reinterpret_cast<__nv_bfloat162*>(y) = __floats2bfloat162_rn(v[0], v[1]);
                else
                    for (int e = 0; e < STEP && col + e < p.outs; ++e) y[e] = __float2bfloat16_rn(v[e]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(BN));
}

// ---- few rows: a cached token of a serving batch --------------------------------------------------------------------
// Bound by the weight, read once, and behind that by the latency of one launch.  Two CTAs of eight warps per SM stay for
// all their tiles of 8 CG weight rows (gate and value rows side by side with SwiGLU).  A warp takes one group of eight
// weight rows and a slice of K; a lane keeps the 16-byte pieces of three steps in flight ahead of the products.  The products
// run on mma.sync m16n8k32 with the rows of x as the M side: the contraction index is permuted so that a lane's 16-byte
// piece of a weight row is its B fragment of two instructions, and the rows, in shared memory, are read with the same
// permutation.  BF16 rows are quantised by every CTA on the way into shared memory.
constexpr int I8_TOKEN_ROWS = 16;   // past that the tensor-memory kernels take less (24 x 1024 x 7488: 7.6 us against 9.8)
constexpr size_t I8_TOKEN_SMEM = 190 * 1024;
constexpr int I8_TOKEN_BATCH = 4, I8_TOKEN_AHEAD = 3;   // weight pieces per lane and step, steps in flight
// Row pitch in shared memory, 64 bytes off a multiple of 128: the eight 16-byte pieces a quarter-warp reads (two rows, four
// consecutive pieces) fall into distinct banks.
__host__ __device__ constexpr long long int8_pitch(int K) { return ((long long)K + 127) / 128 * 128 + 64; }

struct Int8TokenParams {
    Int8Params o;              // M, outs, K, scales, bias, y
    const void* x;             // rows, x_stride elements apart, on 16-byte boundaries; K a multiple of eight in BF16
    long long x_stride;
    const signed char* W;      // [N][w_stride], readable up to K rounded up to 16
    long long w_stride;
};

__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A 16-byte piece of a weight row: read once by one CTA, and ahead of the wait for the kernel before.
__device__ __forceinline__ uint4 load_weight(const signed char* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

// The rows of x as int8 in shared memory, zeros past K; T: BF16 rows are quantised, int8 rows are copied.
template <class T>
__device__ __forceinline__ void int8_rows(const Int8TokenParams& p, signed char* s_q, float* s_scale, unsigned* s_top) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, M = p.o.M, K = p.o.K;
    const int pitch = (int)int8_pitch(K);
    if constexpr (sizeof(T) == 1) {
        const int pieces = pitch / 16;   // asynchronous copies: all rows in flight at once, what lies past K comes as zeros
        for (int idx = tid; idx < M * pieces; idx += 256) {
            const int m = idx / pieces, c0 = (idx - m * pieces) * 16, n = min(16, max(0, K - c0));
            const signed char* from = reinterpret_cast<const signed char*>(p.x) + m * p.x_stride + (n > 0 ? c0 : 0);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc_smem(s_q + (long long)m * pitch + c0)), "l"(from), "r"(n) : "memory");
        }
        asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        if (tid < M) s_scale[tid] = p.o.x_scale[tid];
    } else {
        // units of 256 entries of a row, a warp each; the first HELD of a warp stay in registers between the two passes
        constexpr int HELD = 4;
        const int segs = (pitch + 255) / 256, units = M * segs;
        const auto unit = [&](int u) {
            const int m = u / segs;
            return load_piece<T, true>(reinterpret_cast<const T*>(p.x) + m * p.x_stride, u < units ? (u - m * segs) * 256 + lane * 8 : K, K);
        };
        const auto widen = [&](int u, const Piece<T>& piece) {
            if (u >= units) return;
            const unsigned top = __reduce_max_sync(0xffffffffu, whole_top<T>(piece_top(piece, 0)));
            if (lane == 0) atomicMax(s_top + u / segs, top);
        };
        const auto store = [&](int u, const Piece<T>& piece) {
            if (u >= units) return;
            const int m = u / segs, c0 = (u - m * segs) * 256 + lane * 8;
            const RowScale r = row_scale(s_top[m]);
            if (c0 < pitch) *reinterpret_cast<uint2*>(s_q + (long long)m * pitch + c0) = quantize_piece(piece, r);
            if (c0 == 0) s_scale[m] = r.scale;
        };
        Piece<T> held[HELD];
#pragma unroll
        for (int h = 0; h < HELD; ++h) held[h] = unit(warp + 8 * h);
        if (tid < M) s_top[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) widen(warp + 8 * h, held[h]);
        for (int u = warp + 8 * HELD; u < units; u += 8) widen(u, unit(u));
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) store(warp + 8 * h, held[h]);
        for (int u = warp + 8 * HELD; u < units; u += 8) store(u, unit(u));
    }
}

// RG: groups of eight rows; CG: groups of eight weight rows per CTA (2 with GATED)
template <int RG, int CG, bool GATED, class T>
__global__ void __launch_bounds__(256, 2) k_int8_token(Int8TokenParams p) {
    static_assert(!GATED || CG == 2, "gate and value rows are the two groups");
    constexpr int KS = 8 / CG, MT = (RG + 1) / 2, B = I8_TOKEN_BATCH;
    extern __shared__ __align__(16) unsigned char i8_raw[];
    signed char* s_q = reinterpret_cast<signed char*>(i8_raw);
    __shared__ int s_red[2][8][RG * 8][9];
    __shared__ float s_scale[RG * 8];
    __shared__ unsigned s_top[RG * 8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int cg = warp % CG, ks = warp / CG, M = p.o.M, K = p.o.K, outs = p.o.outs;
    constexpr int WIDTH = GATED ? 8 : 8 * CG;
    const int tiles = (outs + WIDTH - 1) / WIDTH;
    const int chunks = (K + 63) / 64, per = (chunks + KS - 1) / KS;
    const int begin = min(ks * per, chunks), end = min(begin + per, chunks);
    const int steps = (per + B - 1) / B;
    const int pitch = (int)int8_pitch(K);

    // The next step to be requested: its tile, its number there, and its first pieces.  (Counted on; a division per step was a
    // third of the instructions.)
    int want_tile = blockIdx.x, want_step = 0;
    const signed char* want = nullptr;
    bool want_live = false;
    const auto request = [&](uint4 (&w)[B]) {
        if (want_step == 0) {
            const int col = want_tile * WIDTH + (GATED ? g : cg * 8 + g);
            want_live = want_tile < tiles && col < outs;
            want = p.W + (long long)(GATED ? col + cg * outs : col) * p.w_stride + begin * 64 + t * 16;
        }
        const int base = begin + want_step * B;
#pragma unroll
        for (int i = 0; i < B; ++i)
            w[i] = want_live && base + i < end && (base + i) * 64 + t * 16 < K ? load_weight(want + i * 64) : make_uint4(0u, 0u, 0u, 0u);
        want += B * 64;
        if (++want_step == steps) {
            want_step = 0;
            want_tile += gridDim.x;
        }
    };
    uint4 w[I8_TOKEN_AHEAD][B];
#pragma unroll
    for (int i = 0; i < I8_TOKEN_AHEAD; ++i) request(w[i]);
    chain_wait();
    chain_release();
    int8_rows<T>(p, s_q, s_scale, s_top);
    __syncthreads();

    // the columns that a thread finishes are the same ones of every tile
    const int out_col = tid % WIDTH;
    float scale[2], bias[2];
    const auto finish_of = [&](int tile) {
        const int n = tile * WIDTH + out_col;
#pragma unroll
        for (int j = 0; j < (GATED ? 2 : 1); ++j) {
            scale[j] = n < outs ? p.o.w_scale[n + j * outs] : 0.f;
            bias[j] = n < outs ? int8_bias(p.o, n + j * outs) : 0.f;
        }
    };
    int acc[MT][4];
    int tile = blockIdx.x, st = 0, buf = 0;
    const auto step = [&](uint4 (&w)[B]) {
        const int base = begin + st * B;
        if (st == 0) {
            finish_of(tile);   // requested ahead of the products
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[a][e] = 0;
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (base + i < end) {   // warp-uniform
                const signed char* sx = s_q + (base + i) * 64 + t * 16;
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    const int r0 = a * 16 + g, r1 = r0 + 8;
                    const uint4 lo = r0 < M ? *reinterpret_cast<const uint4*>(sx + r0 * pitch) : make_uint4(0u, 0u, 0u, 0u);
                    const uint4 hi = 2 * a + 1 < RG && r1 < M ? *reinterpret_cast<const uint4*>(sx + r1 * pitch) : make_uint4(0u, 0u, 0u, 0u);
                    mma_s8(acc[a], lo.x, hi.x, lo.y, hi.y, w[i].x, w[i].y);
                    mma_s8(acc[a], lo.z, hi.z, lo.w, hi.w, w[i].z, w[i].w);
                }
            }
        }
        request(w);
        if (++st != steps) return;
        // last step of a tile: the K slices are added up through shared memory (two buffers in turn, so one barrier)
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            s_red[buf][warp][a * 16 + g][2 * t] = acc[a][0];
            s_red[buf][warp][a * 16 + g][2 * t + 1] = acc[a][1];
            if (2 * a + 1 < RG) {
                s_red[buf][warp][a * 16 + 8 + g][2 * t] = acc[a][2];
                s_red[buf][warp][a * 16 + 8 + g][2 * t + 1] = acc[a][3];
            }
        }
        __syncthreads();
        const int n = tile * WIDTH + out_col;
        for (int m = tid / WIDTH; m < M && n < outs; m += 256 / WIDTH) {
            const auto value = [&](int group, int j) {
                int v = 0;
#pragma unroll
                for (int k = 0; k < KS; ++k) v += s_red[buf][k * CG + group][m][out_col & 7];
                return (float)v * s_scale[m] * scale[j] + bias[j];
            };
            float out = value(GATED ? 0 : out_col >> 3, 0);
            if constexpr (GATED) out = int8_gated(out, value(1, 1));
            if (p.o.out_f32) reinterpret_cast<float*>(p.o.y)[m * p.o.y_stride + n] = out;
            else reinterpret_cast<__nv_bfloat16*>(p.o.y)[m * p.o.y_stride + n] = __float2bfloat16_rn(out);
        }
        st = 0;
        buf ^= 1;
        tile += gridDim.x;
    };
    while (tile < tiles) {
#pragma unroll
        for (int i = 0; i < I8_TOKEN_AHEAD; ++i)
            if (tile < tiles) step(w[i]);
    }
}

}  // namespace sd
