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
// A row is kept in shared memory by a cluster of C CTAs, contiguous slices of the vocabulary, a contiguous range a warp.
// A rule first takes a histogram of the row over 1024 equal steps of (x_max - x) / T, of counts (top-k) or of weights to 16
// bits (top-p), which says in which step its border lies at most.  What is in front of that is all that can be drawn:
// * up to 512 candidates go to the first CTA, one a thread, which sorts them, sums them up and draws;
// * more are moved together by their warps, in place.  The exact border comes from a histogram over them and from further
//   ones, over equal steps of the logit's bits, until one value is left; sums and draw go over what was moved.
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
constexpr int SAMPLE_GROUPS = SAMPLE_BINS / 32;   // of 32 bins, summed by every CTA for itself
static_assert(SAMPLE_GROUPS == 32 && SAMPLE_GROUPS == 2 * SAMPLE_WARPS, "a lane each, two a warp");
constexpr int SAMPLE_WEIGHT_BITS = 44;
constexpr int SAMPLE_RANGE = 45;          // binades under the largest weight that are not rounded to zero
constexpr int SAMPLE_TABLE = 128;         // steps of a binade in the exponential's table
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
    double power[SAMPLE_TABLE];   // 2^(j / SAMPLE_TABLE)
    unsigned count[SAMPLE_BINS];
    u64 mass[SAMPLE_BINS];
    u64 group_mass[SAMPLE_GROUPS];
    unsigned group_count[SAMPLE_GROUPS];
    u64 warp_sum[SAMPLE_WARPS];
    unsigned warp_eq[SAMPLE_WARPS];
    float warp_max[SAMPLE_WARPS];
    float top;                    // largest logit of the slice
    u64 total_gt;                 // of the slice: weight (above the border), candidates on the border
    unsigned total_eq;
    unsigned kept;                // of the slice: entries in front of the border (written once)
    unsigned low, high;           // of the slice: smallest and largest bits in a step
    int bin;
    unsigned bin_count;
    u64 before;
};

// 2^(44 - t) to the nearest whole number, t in steps of 1 / 128 binade, 0 <= t < 45 * 128: with n the whole number next to
// -t, 2^(n / 128) from a table and an exponent, and 2^(r / 128) for the rest |r| <= 1/2 from the exponential's series, cut
// behind the fourth power (the term left out is below 2^-49).  Table-driven exponential: P. T. P. Tang, ACM TOMS 15 (1989).
__device__ __forceinline__ u64 fixed_power(double t, const double* table) {
    constexpr double ROUND = 6755399441055744.0;   // 1.5 * 2^52: a sum with it is rounded to a whole number
    constexpr double L = 0.693147180559945309417 / SAMPLE_TABLE;
    const double shifted = ROUND - t;
    const double r = (ROUND - shifted) - t;
    const int n = __double2loint(shifted);
    double e = fma(r, L * L * L * L / 24, L * L * L / 6);
    e = fma(r, e, L * L / 2);
    e = fma(r, e, L);
    e = fma(r, e, 1.0);
    const double p = table[n & (SAMPLE_TABLE - 1)];
    const double scaled = __hiloint2double(__double2hiint(p) + (((n >> 7) + SAMPLE_WEIGHT_BITS) << 20), __double2loint(p));
    return (u64)__double_as_longlong(fma(e, scaled, 0x1p52)) - (u64)__double_as_longlong(0x1p52);
}
static_assert(SAMPLE_TABLE == 128, "fixed_power shifts by seven bits");

template <class T, int C>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) k_sample(SampleParams p) {
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
    T* const mine = s_x + v0 * VE;        // the warp's range
    int held = (v1 - v0) * VE;            // and how many entries it still holds
    const auto load = [&](int v, T (&e)[VE]) {
        const int at = first + v * VE - shift;   // index of the vector's first element in the row
        if (at >= 0 && at + VE <= p.V) {
            *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(x + at);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) e[j] = at + j >= 0 && at + j < p.V ? x[at + j] : T(-INFINITY);
        }
    };

    float top = -INFINITY;
#pragma unroll 4
    for (int v = v0 + lane; v < v1; v += 32) {
        alignas(16) T e[VE];
        load(v, e);
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
    if (tid < SAMPLE_TABLE) sh.power[tid] = exp2((double)tid / SAMPLE_TABLE);
    for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.count[b] = 0;
    __syncthreads();
    top = sh.warp_max[lane & (SAMPLE_WARPS - 1)];
#pragma unroll
    for (int s = SAMPLE_WARPS / 2; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if constexpr (C > 1) {
        if (tid == 0) sh.top = top;
        everywhere();
#pragma unroll
        for (int r = 0; r < C; ++r) top = fmaxf(top, *of_rank(&sh.top, r));
    }

    if (top == -INFINITY) {   // nothing to draw
        if (rank == 0 && tid == 0) p.tokens[row] = p.empty_token;
        everywhere();         // no CTA leaves while another may read its memory
        return;
    }
    const bool infinite = top == INFINITY;
    if (infinite) {           // infinite logits share the draw: they become zeros, everything else is out
        for (int i = lane; i < held; i += 32) mine[i] = to_float(mine[i]) == INFINITY ? T(0.f) : T(-INFINITY);
        __syncwarp();
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
    temperature = fmin(temperature, 1e30);   // differences of logits that leave FP32 weigh nothing at any temperature
    const double slope = 1.4426950408889634 * SAMPLE_TABLE / temperature;      // table steps per unit of logit
    const float bin_slope = (float)(slope * ((double)SAMPLE_BINS / (SAMPLE_RANGE * SAMPLE_TABLE)));
    const double reach = min_p > 0.0 ? fmax(0.0, -log2(min_p)) * SAMPLE_TABLE : INFINITY;   // table steps that min-p leaves
    const auto steps_below = [&](float v) { return ((double)top - (double)v) * slope; };
    const auto weight = [&](float v) -> u64 {
        const double t = steps_below(v);
        return t < (double)(SAMPLE_RANGE * SAMPLE_TABLE) ? fixed_power(t, sh.power) : 0ull;
    };
    const auto bin_of = [&](float v) { return min(SAMPLE_BINS - 1, __float2int_rz((top - v) * bin_slope)); };

    // Every vector of a warp's range, before anything is moved.
    const auto each_loaded = [&](auto&& f) {
        for (int v = v0 + lane; v < v1; v += 32) {
            const uint4 raw = *reinterpret_cast<const uint4*>(s_x + v * VE);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int j = 0; j < VE; ++j) f(to_float(e[j]));
        }
    };
    // Every entry that is left.
    const auto each = [&](auto&& f) {
        for (int i = lane; i < held; i += 32) f(to_float(mine[i]));
    };
    const auto block_sum = [&](u64 v) {   // over the slice, to total_gt
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
        if (lane == 0) sh.warp_sum[warp] = v;
        __syncthreads();
        if (tid == 0) {
            u64 a = 0;
            for (int w = 0; w < SAMPLE_WARPS; ++w) a += sh.warp_sum[w];
            sh.total_gt = a;
        }
    };
    // The sums of the CTA's groups of bins, then a barrier of the row: what find() reads.
    const auto publish = [&](bool counts, bool masses) {
        __syncthreads();
#pragma unroll
        for (int g = 2 * warp; g < 2 * warp + 2; ++g) {
            if (counts) {
                const unsigned c = __reduce_add_sync(0xffffffffu, sh.count[g * 32 + lane]);
                if (lane == 0) sh.group_count[g] = c;
            }
            if (masses) {
                u64 m = sh.mass[g * 32 + lane];
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) m += __shfl_xor_sync(0xffffffffu, m, s);
                if (lane == 0) sh.group_mass[g] = m;
            }
        }
        everywhere();
    };
    // The bin of which `hit` says, by the running sum before and behind it, that it is the one (-1: none), with its entries and
    // the sum before it.  of(bins) and of(groups) give a lane's sum of the whole row.  The first warp looks, groups first:
    // reading every bin of every CTA took 5 us.
    const auto find = [&](u64 carried, auto&& group_sum, auto&& bin_sum, auto&& hit) {
        if (warp == 0) {
            int found = -1;
            u64 before = carried;
            unsigned entries = 0;
#pragma unroll
            for (int level = 0; level < 2; ++level) {
                const int at = level == 0 ? lane : found * 32 + lane;
                const u64 own = level == 0 ? group_sum(at) : bin_sum(at);
                u64 sum = own;
#pragma unroll
                for (int s = 1; s < 32; s <<= 1) {
                    const u64 o = __shfl_up_sync(0xffffffffu, sum, s);
                    if (lane >= s) sum += o;
                }
                sum += before;
                const unsigned who = __ballot_sync(0xffffffffu, hit(sum - own, sum));
                if (who == 0) {
                    found = -1;
                    break;
                }
                const int l = __ffs(who) - 1;
                found = level == 0 ? l : found * 32 + l;
                before = __shfl_sync(0xffffffffu, sum - own, l);
            }
            if (found >= 0 && lane < C) entries = *of_rank(&sh.count[found], lane);
            entries = __reduce_add_sync(0xffffffffu, entries);
            if (lane == 0) {
                sh.bin = found;
                sh.before = before;
                sh.bin_count = entries;
            }
        }
        everywhere();   // found, and no CTA clears what another still reads
    };
    const auto group_counts = [&](int g) {
        u64 c = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) c += *of_rank(&sh.group_count[g], r);
        return c;
    };
    const auto counts = [&](int b) {
        u64 c = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) c += *of_rank(&sh.count[b], r);
        return c;
    };
    const auto group_masses = [&](int g) {
        u64 m = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) m += *of_rank(&sh.group_mass[g], r);
        return m;
    };
    const auto masses = [&](int b) {
        u64 m = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) m += *of_rank(&sh.mass[b], r);
        return m;
    };
    const auto clear = [&]() {
        for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
            sh.count[b] = 0;
            sh.mass[b] = 0;
        }
        __syncthreads();
    };
    // Which entries of a vector lie in the bins up to `bin`.
    const auto in_front = [&](const T (&e)[VE], int bin) {
        unsigned stays = 0;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const float f = to_float(e[j]);
            if (f > -INFINITY && bin_of(f) <= bin) stays |= 1u << j;   // a NaN is not
        }
        return stays;
    };
    const auto prefix = [&](int n, int& all) {   // over the lanes in front
        int upto = n;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, s);
            if (lane >= s) upto += o;
        }
        all = __shfl_sync(0xffffffffu, upto, 31);
        return upto - n;
    };
    // Walks over the warp's range: f(vector, its entries up to `bin`, how many of them are in front of the vector's).
    const auto walk = [&](int bin, auto&& f) {
        int kept = 0;
        for (int base = v0; base < v1; base += 32) {
            const int v = base + lane;
            alignas(16) T e[VE];
            unsigned stays = 0;
            if (v < v1) {
                *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(s_x + v * VE);
                stays = in_front(e, bin);
            }
            int all;
            const int at = kept + prefix(__popc(stays), all);
            f(v, e, stays, at);
            kept += all;
            __syncwarp();
        }
        return kept;
    };
    int last = SAMPLE_BINS;   // the last bin that was kept
    // Counts what lies in the bins up to `bin`.  Few entries go to the first CTA: true, and sh.mass there holds their keys
    // (ordered by logit, then by place), sh.count their indices.  More move to the front of their warp's range, in order.
    unsigned listed = 0;
    const auto keep_up_to = [&](int bin) {
        last = bin;
        unsigned n = 0;
        for (int v = v0 + lane; v < v1; v += 32) {
            alignas(16) T e[VE];
            *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(s_x + v * VE);
            n += __popc(in_front(e, bin));
        }
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) sh.warp_eq[warp] = n;
        __syncthreads();
        unsigned in_warps = lane < SAMPLE_WARPS ? sh.warp_eq[lane] : 0;
        const unsigned before_warp = __reduce_add_sync(0xffffffffu, lane < warp ? in_warps : 0);
        in_warps = __reduce_add_sync(0xffffffffu, in_warps);
        if (tid == 0) sh.kept = in_warps;
        everywhere();
        const unsigned in_slices = lane < C ? *of_rank(&sh.kept, lane) : 0;
        const unsigned before_slice = __reduce_add_sync(0xffffffffu, lane < rank ? in_slices : 0);
        listed = __reduce_add_sync(0xffffffffu, in_slices);
        if (listed > SAMPLE_THREADS) {
            held = walk(bin, [&](int, const T (&e)[VE], unsigned stays, int at) {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < VE; ++j)
                    if (stays >> j & 1) mine[at++] = e[j];   // never ahead of what the warp has read
            });
            return false;
        }
        u64* keys = of_rank(sh.mass, 0);
        unsigned* indices = of_rank(sh.count, 0);
        walk(bin, [&](int v, const T (&e)[VE], unsigned stays, int at) {
            unsigned place = before_slice + before_warp + at;
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (stays >> j & 1) {
                    keys[place] = (u64)order_bits(to_float(e[j])) << 32 | (0xffffffffu - place);
                    indices[place++] = first + v * VE + j - shift;
                }
        });
        everywhere();
        return true;
    };
    const auto block_scan = [&](u64 v, u64& all) {   // sum of the threads up to this one, and of all
        u64 sum = v;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const u64 o = __shfl_up_sync(0xffffffffu, sum, s);
            if (lane >= s) sum += o;
        }
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = sum;
        __syncthreads();
        all = 0;
        for (int w = 0; w < SAMPLE_WARPS; ++w) {
            if (w < warp) sum += sh.warp_sum[w];
            all += sh.warp_sum[w];
        }
        return sum;
    };
    const auto uniform_part = [&](u64 all) {   // the whole part of u times the sum
        const float u = p.uniform[row];
        const double clipped = u > 0.f ? fmin((double)u, 1.0 - 0x1p-53) : 0.0;   // a NaN counts as zero
        return __umul64hi(all, (u64)(clipped * 0x1p64));
    };
    // The rest of the row's work where few candidates are left, by the first CTA: one a thread, sorted by logit and place.
    const auto draw_from_list = [&](unsigned k, bool by_p, double target, bool sum_first) {
        if (rank != 0) return;
        u64 key = tid < (int)listed ? sh.mass[tid] : 0ull;
        if (k < listed || by_p) {
            for (int size = 2; size < 2 * (int)listed; size <<= 1)
                for (int j = size >> 1; j > 0; j >>= 1) {
                    u64 other;
                    if (j >= 32) {
                        __syncthreads();
                        sh.mass[tid] = key;
                        __syncthreads();
                        other = sh.mass[tid ^ j];
                    } else {
                        other = __shfl_xor_sync(0xffffffffu, key, j);
                    }
                    const bool larger = ((tid & size) == 0) == ((tid & j) == 0);
                    if (larger ? other > key : other < key) key = other;
                }
        }
        const unsigned place = 0xffffffffu - (unsigned)key;
        const float v = from_order_bits((unsigned)(key >> 32));
        const double t = steps_below(v);
        const u64 w = tid < (int)listed && tid < (int)k && t < (double)(SAMPLE_RANGE * SAMPLE_TABLE) ? fixed_power(t, sh.power) : 0ull;
        bool stays = w != 0 && t <= reach;
        if (by_p) {
            u64 all;
            const u64 upto = block_scan(w, all);
            if (sum_first) target = top_p * (double)all;
            stays = stays && (double)(upto - w) < target;
        }
        __syncthreads();
        sh.mass[tid] = 0;
        __syncthreads();
        if (stays) sh.mass[place] = w;
        __syncthreads();
        const u64 own = sh.mass[tid];
        u64 all;
        const u64 upto = block_scan(own, all), drawn = uniform_part(all);
        if (drawn < upto && drawn >= upto - own) p.tokens[row] = sh.count[tid];
    };

    // what stays: logits above `edge`, and the first `ties` of those on it
    float edge = -INFINITY;
    unsigned ties = 0, on_edge = 0;

    // The border inside the bin that sh.bin names, among entries of which in_bin says whether they are in it.  By weight, a
    // running sum reaches `target`; by count, it reaches `count`.
    const auto refine = [&](bool by_mass, unsigned count, double target) {
        const int bin = sh.bin;
        unsigned low = 0xffffffffu, high = 0;
        each([&](float v) {
            if (bin_of(v) != bin || !(v > -INFINITY) || v < edge) return;
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
            const u64 carried = sh.before;
            clear();
            each([&](float v) {
                const unsigned k = order_bits(v);
                if (k < low || k > high) return;
                const int b = (int)((high - k) >> down);
                if (by_mass) {
                    const u64 w = weight(v);
                    if (w == 0) return;
                    atomicAdd(&sh.mass[b], w);
                }
                atomicAdd(&sh.count[b], 1u);
            });
            publish(true, by_mass);
            if (by_mass)
                find(carried, group_masses, masses, [&](u64 a, u64 b) { return (double)a < target && !((double)b < target); });
            else
                find(carried, group_counts, counts, [&](u64 a, u64 b) { return a < count && b >= count; });
            high -= (unsigned)sh.bin << down;
            low = down == 0 ? high : max(low, high - ((1u << down) - 1));
        }
        edge = from_order_bits(high);
        on_edge = sh.bin_count;
        if (by_mass) {
            const u64 w = weight(edge), before = sh.before;
            unsigned keep = 1;
            const double want = (target - (double)before) / (double)w;
            if (want > 1.0) keep = (unsigned)fmin(ceil(want), (double)on_edge);
            while (keep > 1 && !((double)(before + (keep - 1) * w) < target)) --keep;
            while (keep < on_edge && (double)(before + keep * w) < target) ++keep;
            ties = keep;
        } else {
            ties = count - (unsigned)sh.before;
        }
        __syncthreads();   // sh.before and sh.bin_count are read by everyone before they change
    };

    const int min_p_bin = reach < SAMPLE_RANGE * SAMPLE_TABLE ? (int)(reach * ((double)SAMPLE_BINS / (SAMPLE_RANGE * SAMPLE_TABLE))) + 1 : SAMPLE_BINS;
    const bool by_k = top_k > 1 && top_k < p.V, by_p = top_k != 1 && top_p < 1.0;
    double target = 0.0;
    if (top_k == 1) {
        // the first entry that equals the largest
        unsigned at = 0xffffffffu;
        for (int v = v0 + lane; v < v1; v += 32) {
            const uint4 raw = *reinterpret_cast<const uint4*>(s_x + v * VE);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int j = VE - 1; j >= 0; --j)
                if (to_float(e[j]) == top) at = min(at, (unsigned)(first + v * VE + j - shift));
        }
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) sh.warp_eq[warp] = at;
        __syncthreads();
        if (warp == 0) {
            at = __reduce_min_sync(0xffffffffu, sh.warp_eq[lane & (SAMPLE_WARPS - 1)]);
            if (lane == 0) sh.low = at;
        }
        everywhere();
        if (rank == 0 && warp == 0) {
            at = __reduce_min_sync(0xffffffffu, *of_rank(&sh.low, lane & (C - 1)));
            if (lane == 0) p.tokens[row] = at;
        }
        everywhere();   // no CTA leaves while another may read its memory
        return;
    }
    if (by_k) {
        each_loaded([&](float v) {
            if (v > -INFINITY) atomicAdd(&sh.count[bin_of(v)], 1u);
        });
        publish(true, false);
        find(0, group_counts, counts, [&](u64 a, u64 b) { return a < (unsigned)top_k && b >= (unsigned)top_k; });
        const int bin = sh.bin;   // -1: fewer candidates than top-k keeps
        const int limit = bin < 0 ? SAMPLE_BINS - 1 : bin;
        const bool cut = !by_p && min_p_bin < limit;   // by min-p: all that is in front of that is among the first k
        if (keep_up_to(cut ? min_p_bin : limit)) {
            draw_from_list((unsigned)top_k, by_p, 0.0, true);
            return;
        }
        if (!cut && bin >= 0) refine(false, (unsigned)top_k, 0.0);
        if (by_p) {   // the weight of what top-k keeps
            u64 sum = 0;
            each([&](float v) { if (v > edge) sum += weight(v); });
            block_sum(sum);
            everywhere();
            u64 all = edge > -INFINITY ? ties * weight(edge) : 0ull;
            for (int r = 0; r < C; ++r) all += *of_rank(&sh.total_gt, r);
            target = top_p * (double)all;
        }
    } else if (by_p) {
        // the sum of all weights, and a histogram of their upper 16 bits (relative to the largest of the bin): its running
        // sums are not above the true ones, so the border is not behind the bin in which they reach the target
        const auto bin_shift = [](int b) { return max(0, SAMPLE_WEIGHT_BITS - 15 - b * SAMPLE_RANGE / SAMPLE_BINS); };
        u64 sum = 0;
        each_loaded([&](float v) {
            const u64 w = weight(v);
            sum += w;
            const int b = bin_of(v);
            if (w != 0) atomicAdd(&sh.count[b], (unsigned)(w >> bin_shift(b)));
        });
        block_sum(sum);
        for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.mass[b] = (u64)sh.count[b] << bin_shift(b);
        publish(false, true);
        u64 all = 0;
        for (int r = 0; r < C; ++r) all += *of_rank(&sh.total_gt, r);
        target = top_p * (double)all;
        find(0, group_masses, masses, [&](u64 a, u64 b) { return (double)a < target && !((double)b < target); });
        if (keep_up_to(min(sh.bin < 0 ? SAMPLE_BINS - 1 : sh.bin, min_p_bin))) {
            draw_from_list(SAMPLE_THREADS, true, target, false);
            return;
        }
    } else if (min_p_bin < SAMPLE_BINS) {
        if (keep_up_to(min_p_bin)) {
            draw_from_list(SAMPLE_THREADS, false, 0.0, false);
            return;
        }
    }
    if (by_p) {
        clear();
        each([&](float v) {
            const u64 w = weight(v);
            if (w == 0 || v < edge) return;
            const int b = bin_of(v);
            atomicAdd(&sh.mass[b], w);
            atomicAdd(&sh.count[b], 1u);
        });
        publish(true, true);
        find(0, group_masses, masses, [&](u64 a, u64 b) { return (double)a < target && !((double)b < target); });
        if (sh.bin >= 0) refine(true, 0, target);   // else min-p has cut in front of the border
    }

    // the draw
    const auto drawn_weight = [&](float v) -> u64 {
        const double t = steps_below(v);
        return t <= reach && t < (double)(SAMPLE_RANGE * SAMPLE_TABLE) ? fixed_power(t, sh.power) : 0ull;
    };
    const u64 edge_weight = edge > -INFINITY ? drawn_weight(edge) : 0ull;
    u64 gt = 0;
    unsigned eq = 0;
    each([&](float v) {
        if (v > edge) gt += drawn_weight(v);
        else if (v == edge) ++eq;
    });
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) sh.warp_eq[warp] = eq;
    block_sum(gt);
    if (tid == 0) {
        unsigned b = 0;
        for (int w = 0; w < SAMPLE_WARPS; ++w) b += sh.warp_eq[w];
        sh.total_eq = b;
    }
    everywhere();
    u64 all = 0, before = 0, own = 0;
    unsigned seen = 0, passed = 0;   // candidates on the edge before this slice, then before this warp
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
    everywhere();   // the last access to another CTA's memory
    const u64 drawn = uniform_part(all);
    if (drawn < before || drawn >= before + own) return;   // another slice's
    for (int w = 0; w < warp; ++w) {
        const unsigned e = sh.warp_eq[w], keep = seen < ties ? min(e, ties - seen) : 0;
        before += sh.warp_sum[w] + keep * edge_weight;
        seen += e;
    }
    own = sh.warp_sum[warp] + (seen < ties ? min(sh.warp_eq[warp], ties - seen) : 0) * edge_weight;
    if (drawn < before || drawn >= before + own) return;   // another warp's
    int place = -1;   // of the token among what the warp holds
    for (int base = 0; base < held && place < 0; base += 32) {
        const int i = base + lane;
        const float f = i < held ? to_float(mine[i]) : -INFINITY;
        const bool on = f == edge && f > -INFINITY;
        const unsigned edge_lanes = __ballot_sync(0xffffffffu, on);
        u64 sum = f > edge ? drawn_weight(f) : on && seen + __popc(edge_lanes & ((1u << lane) - 1)) < ties ? edge_weight : 0ull;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const u64 o = __shfl_up_sync(0xffffffffu, sum, s);
            if (lane >= s) sum += o;
        }
        const unsigned over = __ballot_sync(0xffffffffu, before + sum > drawn);
        if (over) place = base + __ffs(over) - 1;
        before += __shfl_sync(0xffffffffu, sum, 31);
        seen += __popc(edge_lanes);
    }
    if (last == SAMPLE_BINS) {   // nothing was moved
        if (lane == 0) p.tokens[row] = first + v0 * VE + place - shift;
        return;
    }
    // the place-th of those entries of the warp's range that were kept, counted again in the row itself
    for (int base = v0; base < v1; base += 32) {
        const int v = base + lane;
        unsigned stays = 0;
        if (v < v1) {
            alignas(16) T e[VE];
            load(v, e);
            if (infinite)
                for (int j = 0; j < VE; ++j) e[j] = to_float(e[j]) == INFINITY ? T(0.f) : T(-INFINITY);
            stays = in_front(e, last);
        }
        int all_kept;
        const int n = __popc(stays), from = prefix(n, all_kept);
        if (place >= from && place < from + n)
            for (int j = 0, k = from; j < VE; ++j)
                if (stays >> j & 1 && k++ == place) p.tokens[row] = first + v * VE + j - shift;
        if (place < all_kept) return;
        place -= all_kept;
    }
}

}  // namespace sd
