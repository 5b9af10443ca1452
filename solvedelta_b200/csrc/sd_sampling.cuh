// One token per row of logits, drawn with temperature, top-k, top-p and min-p from a given uniform number.
//
// The candidates of a row are ordered by logit, ties by index, the lowest first; each has the weight exp((x - x_max) / T).
//   top-k   the first k of the order stay
//   top-p   of those, one stays while the weights before it sum to less than p times the sum of all
//   min-p   of those, one stays if its weight is at least m (x_max has weight 1)
// and the token is the first index, in the order of the vocabulary, at which the running sum of what stays exceeds u times
// the whole.
//
// Weights are 64-bit fixed point, 2^44 for x_max, rounded from an exponential in 64 bits: sums of up to 2^18 of them are
// exact whatever their order, so results depend neither on the split of a row nor on the order of atomics, and a drawn
// index differs from that of real numbers only where u is within about 1e-11 of a border.  A weight under 2^-45 is zero.
//
// A row is kept in shared memory by a cluster of C CTAs, contiguous slices of the vocabulary.  Thresholds come from
// histograms, first of 1024 equal steps of (x_max - x) / T over the 45 binades that carry weight, then, inside the step in
// which the k-th candidate or the p-th part of the weight lies, of equal steps of the logit's bits until one value is left.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "sd_int8.cuh"   // to_float

namespace sd {

struct SampleParams {
    int V;
    const void* logits;
    long long stride;          // elements
    const float* uniform;      // [rows]
    // per row where the pointer is set, else the value
    const float* temperature_row;
    const int* top_k_row;
    const float* top_p_row;
    const float* min_p_row;
    double temperature, top_p, min_p;
    int top_k;
    long long empty_token;
    long long* tokens;
    int slice;                 // elements of a CTA's slice, a multiple of 16 bytes
};

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32, SAMPLE_BINS = 2 * SAMPLE_THREADS;
constexpr int SAMPLE_WEIGHT_BITS = 44;
constexpr double SAMPLE_RANGE = 45.0;     // binades under the largest weight that are not rounded to zero
constexpr int SAMPLE_MAX_VOCAB = 1 << 18;
typedef unsigned long long u64;

// Order-preserving bits of a float, and back.
__device__ __forceinline__ unsigned order_bits(float x) {
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_bits(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct SampleShared {
    unsigned count[SAMPLE_BINS];
    u64 mass[SAMPLE_BINS];
    u64 warp_sum[SAMPLE_WARPS];
    unsigned warp_eq[SAMPLE_WARPS];
    float warp_max[SAMPLE_WARPS];
    float top;                    // largest logit of the slice
    u64 total_gt;                 // of the slice: weight above the threshold, candidates on it
    unsigned total_eq;
    unsigned low, high;           // of the slice: smallest and largest bits in a step
    int bin;
    unsigned bin_count;
    u64 before, total;
};

template <class T, int C>
__global__ void __launch_bounds__(SAMPLE_THREADS) k_sample(SampleParams p) {
    namespace cg = cooperative_groups;
    constexpr int VE = 16 / sizeof(T);
    extern __shared__ __align__(16) unsigned char smp_raw[];
    T* s_x = reinterpret_cast<T*>(smp_raw);
    __shared__ SampleShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / C, rank = blockIdx.x % C;
    const auto everywhere = [&]() {   // a barrier of all CTAs of the row
        if constexpr (C == 1) __syncthreads();
        else cg::this_cluster().sync();
    };
    const auto of_rank = [&](auto* ptr, int r) {
        if constexpr (C == 1) return ptr;
        else return cg::this_cluster().map_shared_rank(ptr, r);
    };
    // The row starts `shift` elements behind a 16-byte boundary; positions count from that boundary, so that the vectors of
    // a slice are aligned in both memories.  Vectors that reach outside the row are read element by element.
    const T* x = reinterpret_cast<const T*>(p.logits) + (long long)row * p.stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int first = rank * p.slice, vectors = max(0, min(p.slice, p.V + shift - first) + VE - 1) / VE;
    const int per_warp = (vectors + SAMPLE_WARPS - 1) / SAMPLE_WARPS, v0 = min(vectors, warp * per_warp), v1 = min(vectors, v0 + per_warp);

    float top = -INFINITY;
    for (int v = v0 + lane; v < v1; v += 32) {
        const int at = first + v * VE - shift;   // index of the vector's first element in the row
        alignas(16) T e[VE];
        if (at >= 0 && at + VE <= p.V) {
            *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(x + at);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) e[j] = at + j >= 0 && at + j < p.V ? x[at + j] : T(-INFINITY);
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const float f = to_float(e[j]);
            if (f != f) e[j] = T(-INFINITY);   // a NaN is never drawn
            else top = fmaxf(top, f);
        }
        *reinterpret_cast<uint4*>(s_x + v * VE) = *reinterpret_cast<const uint4*>(e);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if (lane == 0) sh.warp_max[warp] = top;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < SAMPLE_WARPS; ++w) top = fmaxf(top, sh.warp_max[w]);
        sh.top = top;
    }
    everywhere();
    top = -INFINITY;
#pragma unroll
    for (int r = 0; r < C; ++r) top = fmaxf(top, *of_rank(&sh.top, r));

    if (top == -INFINITY) {   // nothing to draw
        if (rank == 0 && tid == 0) p.tokens[row] = p.empty_token;
        everywhere();         // no CTA leaves while another may read its memory
        return;
    }
    // Every vector of a slice is seen by the thread that loaded it.
    const auto each = [&](auto&& f) {
        for (int v = v0 + lane; v < v1; v += 32) {
            const uint4 raw = *reinterpret_cast<const uint4*>(s_x + v * VE);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int j = 0; j < VE; ++j) f(to_float(e[j]));
        }
    };
    if (top == INFINITY) {    // infinite logits share the draw: they become zeros, everything else is out
        for (int v = v0 + lane; v < v1; v += 32)
            for (int j = 0; j < VE; ++j) s_x[v * VE + j] = to_float(s_x[v * VE + j]) == INFINITY ? T(0.f) : T(-INFINITY);
        top = 0.f;
    }

    double temperature = p.temperature_row ? (double)p.temperature_row[row] : p.temperature;
    const double top_p = p.top_p_row ? (double)p.top_p_row[row] : p.top_p;
    const double min_p = p.min_p_row ? (double)p.min_p_row[row] : p.min_p;
    int top_k = p.top_k_row ? p.top_k_row[row] : p.top_k;
    if (!(temperature > 1e-30) || top_p <= 0.0) {   // the first of the order alone
        top_k = 1;
        temperature = 1.0;
    }
    const double slope = 1.4426950408889634 / temperature;      // binades per unit of logit
    const float bin_slope = (float)(slope * (SAMPLE_BINS / SAMPLE_RANGE));
    const double reach = min_p > 0.0 ? fmax(0.0, -log2(min_p)) : INFINITY;   // binades that min-p leaves
    const auto binades = [&](float v) { return ((double)top - (double)v) * slope; };
    const auto weight_at = [&](double t) -> u64 {
        return t < SAMPLE_RANGE ? (u64)__double2ll_rn(exp2(-t) * (double)(1ull << SAMPLE_WEIGHT_BITS)) : 0ull;
    };
    const auto step_of = [&](float v) { return min(SAMPLE_BINS - 1, __float2int_rz((top - v) * bin_slope)); };

    // what stays so far: logits above `edge`, and the first `ties` of those on it
    float edge = -INFINITY;
    unsigned ties = 0, on_edge = 0;

    // Sums a histogram over the CTAs and finds the bin in which a running sum (of counts, or of weights) reaches the target.
    const auto find = [&](bool by_mass, double fraction, u64 less, unsigned target_count, double& target, bool first_pass) {
        everywhere();   // the histograms are complete
        unsigned c[2] = {0, 0};
        u64 m[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 2; ++j)
            for (int r = 0; r < C; ++r) {
                c[j] += *of_rank(&sh.count[2 * tid + j], r);
                if (by_mass) m[j] += *of_rank(&sh.mass[2 * tid + j], r);
            }
        const u64 mine0 = by_mass ? m[0] : c[0], mine1 = by_mass ? m[1] : c[1];
        u64 sum = mine0 + mine1;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const u64 o = __shfl_up_sync(0xffffffffu, sum, s);
            if (lane >= s) sum += o;
        }
        if (lane == 31) sh.warp_sum[warp] = sum;
        if (tid == 0) sh.bin = -1;
        __syncthreads();
        u64 base = 0, all = 0;
        for (int w = 0; w < SAMPLE_WARPS; ++w) {
            if (w < warp) base += sh.warp_sum[w];
            all += sh.warp_sum[w];
        }
        if (first_pass && by_mass) target = fraction * (double)(all - less);
        const u64 before0 = base + sum - mine0 - mine1 + (first_pass ? 0 : sh.before), before1 = before0 + mine0, after = before1 + mine1;
        __syncthreads();   // sh.before has been read
        const auto reaches = [&](u64 before, u64 upto) {
            return by_mass ? (double)before < target && !((double)upto < target) : before < target_count && upto >= target_count;
        };
        const bool hit0 = reaches(before0, before1), hit1 = reaches(before1, after);
        if (hit0 || hit1) {
            sh.bin = 2 * tid + (hit0 ? 0 : 1);
            sh.bin_count = hit0 ? c[0] : c[1];
            sh.before = hit0 ? before0 : before1;
        }
        everywhere();   // found, and no CTA clears what another still reads
        return sh.bin;
    };
    const auto clear = [&]() {
        for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
            sh.count[b] = 0;
            sh.mass[b] = 0;
        }
        __syncthreads();
    };
    // The threshold of one rule: the first `count` of the order, or those before `fraction` of the weight is reached.
    const auto select = [&](bool by_mass, unsigned count, double fraction) {
        const float old_edge = edge;
        const u64 less = by_mass && edge > -INFINITY ? (u64)(on_edge - ties) * weight_at(binades(edge)) : 0ull;
        double target = 0.0;
        clear();
        each([&](float v) {
            if (v == -INFINITY || v < old_edge) return;
            const int b = step_of(v);
            if (by_mass) {
                const u64 w = weight_at(binades(v));
                if (w == 0) return;
                atomicAdd(&sh.mass[b], w);
            }
            atomicAdd(&sh.count[b], 1u);
        });
        const int bin = find(by_mass, fraction, less, count, target, true);
        if (bin < 0) return;   // fewer candidates than top-k keeps
        // the bits inside the step
        unsigned low = 0xffffffffu, high = 0;
        each([&](float v) {
            if (v == -INFINITY || v < old_edge || step_of(v) != bin) return;
            const unsigned k = order_bits(v);
            low = min(low, k);
            high = max(high, k);
        });
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        if (tid == 0) { sh.low = 0xffffffffu; sh.high = 0; }
        __syncthreads();
        if (lane == 0) { atomicMin(&sh.low, low); atomicMax(&sh.high, high); }
        everywhere();
#pragma unroll
        for (int r = 0; r < C; ++r) {
            low = min(low, *of_rank(&sh.low, r));
            high = max(high, *of_rank(&sh.high, r));
        }
        while (low != high) {
            const int width = 32 - __clz(high - low), down = width > 10 ? width - 10 : 0;   // 1024 bins
            clear();
            each([&](float v) {
                if (v == -INFINITY) return;
                const unsigned k = order_bits(v);
                if (k < low || k > high) return;
                const int b = (int)((high - k) >> down);
                if (by_mass) {
                    const u64 w = weight_at(binades(v));
                    if (w == 0) return;
                    atomicAdd(&sh.mass[b], w);
                }
                atomicAdd(&sh.count[b], 1u);
            });
            const int b = find(by_mass, fraction, less, count, target, false);
            high -= (unsigned)b << down;
            low = down == 0 ? high : max(low, high - ((1u << down) - 1));
        }
        edge = from_order_bits(high);
        if (by_mass) {
            const u64 w = weight_at(binades(edge));
            unsigned keep = 1;
            const double want = (target - (double)sh.before) / (double)w;
            if (want > 1.0) keep = (unsigned)fmin(ceil(want), (double)sh.bin_count);
            while (keep > 1 && !((double)(sh.before + (keep - 1) * w) < target)) --keep;
            while (keep < sh.bin_count && (double)(sh.before + keep * w) < target) ++keep;
            ties = keep;
        } else {
            ties = count - (unsigned)sh.before;
        }
        on_edge = sh.bin_count;
        __syncthreads();   // sh.before and sh.bin_count are read by everyone before they change
    };
    if (top_k == 1) {
        edge = top;
        ties = 1;
    } else {
        if (top_k > 0 && top_k < p.V) select(false, (unsigned)top_k, 0.0);
        if (top_p < 1.0) select(true, 0, top_p);
    }

    // the draw
    const auto weight = [&](float v) -> u64 {
        const double t = binades(v);
        return t <= reach ? weight_at(t) : 0ull;
    };
    const u64 edge_weight = edge > -INFINITY ? weight(edge) : 0ull;
    u64 gt = 0;
    unsigned eq = 0;
    each([&](float v) {
        if (v > edge) gt += weight(v);
        else if (v == edge) ++eq;
    });
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) gt += __shfl_xor_sync(0xffffffffu, gt, s);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        sh.warp_sum[warp] = gt;
        sh.warp_eq[warp] = eq;
    }
    __syncthreads();
    if (tid == 0) {
        u64 a = 0;
        unsigned b = 0;
        for (int w = 0; w < SAMPLE_WARPS; ++w) {
            a += sh.warp_sum[w];
            b += sh.warp_eq[w];
        }
        sh.total_gt = a;
        sh.total_eq = b;
    }
    everywhere();
    u64 all = 0, before = 0, own = 0;
    unsigned seen = 0;   // candidates on the edge before this slice, then before this warp
    {
        unsigned passed = 0;
        for (int r = 0; r < C; ++r) {
            const unsigned e = *of_rank(&sh.total_eq, r), keep = passed < ties ? min(e, ties - passed) : 0;
            const u64 sum = *of_rank(&sh.total_gt, r) + keep * edge_weight;
            if (r == rank) {
                before = all;
                own = sum;
                seen = passed;
            }
            all += sum;
            passed += e;
        }
    }
    everywhere();   // the last access to another CTA's memory
    const float u = p.uniform[row];
    const double clipped = u > 0.f ? fmin((double)u, 1.0 - 0x1p-53) : 0.0;   // a NaN counts as zero
    const u64 target = __umul64hi(all, (u64)(clipped * 0x1p64));
    if (target < before || target >= before + own) return;   // another slice's
    for (int w = 0; w < warp; ++w) {
        const unsigned e = sh.warp_eq[w], keep = seen < ties ? min(e, ties - seen) : 0;
        before += sh.warp_sum[w] + keep * edge_weight;
        seen += e;
    }
    own = sh.warp_sum[warp] + (seen < ties ? min(sh.warp_eq[warp], ties - seen) : 0) * edge_weight;
    if (target < before || target >= before + own) return;   // another warp's
    for (int vbase = v0; vbase < v1; vbase += 32) {
        const int v = vbase + lane;
        u64 mine = 0;
        unsigned e = 0;
        alignas(16) T held[VE];
        if (v < v1) {
            *reinterpret_cast<uint4*>(held) = *reinterpret_cast<const uint4*>(s_x + v * VE);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float f = to_float(held[j]);
                if (f > edge) mine += weight(f);
                else if (f == edge) ++e;
            }
        }
        unsigned e_sum = e;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const unsigned o = __shfl_up_sync(0xffffffffu, e_sum, s);
            if (lane >= s) e_sum += o;
        }
        const unsigned e_before = seen + e_sum - e;
        mine += (e_before < ties ? min(e, ties - e_before) : 0) * edge_weight;
        u64 sum = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const u64 o = __shfl_up_sync(0xffffffffu, sum, s);
            if (lane >= s) sum += o;
        }
        u64 run = before + sum - mine;
        if (target >= run && target < run + mine) {
            unsigned ahead = e_before;
            for (int j = 0; j < VE; ++j) {
                const float f = to_float(held[j]);
                if (f > edge) run += weight(f);
                else if (f == edge && ahead++ < ties) run += edge_weight;
                if (run > target) {
                    p.tokens[row] = first + v * VE + j - shift;
                    break;
                }
            }
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
        seen += __shfl_sync(0xffffffffu, e_sum, 31);
        if (target < before) return;
    }
}

}  // namespace sd
