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
// A row is split over a cluster of C CTAs, contiguous slices of the vocabulary, and over their warps.  Short slices are kept
// in shared memory; of long ones (many rows of a large vocabulary) every pass reads the row again, out of L2, through a ring
// of asynchronous copies.
// A rule first takes a histogram of the row over steps of a 16th of a binade of the weight, of counts (top-k) or of weights to 16
// bits (15 or 14 in long slices; top-p), which says in which step its border lies at most.  What is in front of that is all that can be drawn:
// * up to 512 candidates go to the first CTA, one a thread, which sorts them, sums them up and draws;
// * more are moved together by their warps.  The exact border comes from the entries of its step, gathered, or, where those
//   are more than 512, from further histograms over equal steps of the logit's bits, until one value is left; sums and draw
//   go over what was moved;
// * where that is too much for shared memory, the entries of the border's step alone are moved, and the weights in front of it
//   are summed up once (512 rows of 128000, FP32, N(0, 4), top-p 0.95, 30000 kept of each: 1026 us when every histogram read
//   the row again, 623 with the first form of this).
//
// What bounds it.  One row of 32000 (top-k 50 and top-p: 10 us): a dozen phases of 0.3 to 2 us each, cluster barriers and reads
// of another CTA's memory.  512 rows of 128000 in FP32 (top-p 0.95: 280 us for N(0, 16), 563 for N(0, 4); their 262 MB take
// 40 us): instructions, some 105 for a logit of the former, 70 % of the issue slots (FP64 is a seventh busy).  The largest
// logit and the sum of all weights, without a rule, take 55 of them and 207 us.  At 64 registers a thread some variables live
// in local memory; one instruction of a thousand moves them.
#pragma once
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
    int list;                  // rows that are read again: entries a warp can move together
};

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32, SAMPLE_BINS = 2 * SAMPLE_THREADS;
constexpr int SAMPLE_GROUPS = SAMPLE_BINS / 32;   // of 32 bins, summed by every CTA for itself
static_assert(SAMPLE_GROUPS == 32 && SAMPLE_GROUPS == 2 * SAMPLE_WARPS, "a lane each, two a warp");
constexpr int SAMPLE_WEIGHT_BITS = 44;
constexpr int SAMPLE_RANGE = 45;          // binades under the largest weight that are not rounded to zero
constexpr int SAMPLE_TABLE = 128;         // steps of a binade in the exponential's table
constexpr int SAMPLE_BIN_BITS = 3;        // eight of them are a bin
constexpr float SAMPLE_FAR = 63.9f;       // binades, where the last bin ends
static_assert(int(SAMPLE_FAR * SAMPLE_TABLE) >> SAMPLE_BIN_BITS < SAMPLE_BINS, "bins");
constexpr int SAMPLE_MAX_VOCAB = 1 << 18;
constexpr size_t SAMPLE_STAGED = 94 * 1024;     // bytes of a slice that is kept in shared memory: two CTAs share an SM
// Elements of a slice that is read again: longer rows are shared by more CTAs.
template <class T>
constexpr int SAMPLE_MAX_SLICE = sizeof(T) == 4 ? 90000 : 180000;
// Bits of a weight in the first histogram of top-p, as many as leave a counter of 32 bits room for a slice of equal logits: one
// counts 2^bits, or half a table step more at the end of a binade.  (Few bits miss the border's step more often, and a row that
// does ends with a histogram of whole weights: a batch of 512 rows of 128000, FP32, N(0, 4), top-p 0.95: 522 us with 16,
// 537 with 15, 580 with 14.)
template <class T, bool STAGED>
constexpr int SAMPLE_BIN_WEIGHT_BITS = STAGED ? 16 : sizeof(T) == 4 ? 15 : 14;
template <class T, bool STAGED>
constexpr bool SAMPLE_COUNTERS_HOLD =
    (unsigned long long)(STAGED ? SAMPLE_STAGED / sizeof(T) : SAMPLE_MAX_SLICE<T>) * 129 / 128 << SAMPLE_BIN_WEIGHT_BITS<T, STAGED> < 1ull << 32;
constexpr int SAMPLE_RING = 4;            // vectors a lane has in flight, where the row is read again
constexpr size_t SAMPLE_RING_BYTES = size_t(SAMPLE_THREADS) * 16 * SAMPLE_RING;
typedef unsigned long long u64;
// the kernel's parts share its variables by reference: one that is not inlined would keep them in local memory
#define SAMPLE_INLINE __attribute__((always_inline))

// Order-preserving bits of a float (both zeros have the same), and back.
__device__ __forceinline__ unsigned order_bits(float x) {
    const unsigned b = __float_as_uint(__fadd_rn(x, 0.f));
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_bits(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct SampleShared {
    double power[SAMPLE_TABLE];   // 2^(-j / SAMPLE_TABLE)
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
    unsigned in_step;             // of the slice: entries of the border's step
    int bin;
    unsigned bin_count;
    u64 before;
    float edge;
    unsigned ties;
};

// 2^(44 - (n + r) / 128) to the nearest whole number, |r| little over 1/2, and 0 from n = 45 * 128 on: 2^(-n / 128) from a table
// and an exponent, 2^(-r / 128) from the exponential's series, cut behind the fourth power (the term left out is below 2^-49).
// Table-driven exponential: P. T. P. Tang, ACM TOMS 15 (1989).  A double holds the whole number, and sums of 512 of them.
__device__ __forceinline__ double fixed_power(int n, double r, const double* table) {
    constexpr double L = -0.693147180559945309417 / SAMPLE_TABLE;
    double e = fma(r, L * L * L * L / 24, L * L * L / 6);
    e = fma(r, e, L * L / 2);
    e = fma(r, e, L);
    e = fma(r, e, 1.0);
    const double p = table[n & (SAMPLE_TABLE - 1)];
    const int high = __double2hiint(p) + ((SAMPLE_WEIGHT_BITS - (n >> 7)) << 20);
    const double w = fma(e, __hiloint2double(high, __double2loint(p)), 0x1p52) - 0x1p52;   // rounded by the sum
    return n < SAMPLE_RANGE * SAMPLE_TABLE ? w : 0.0;   // farther entries have no r: they may be infinite
}
static_assert(SAMPLE_TABLE == 128, "fixed_power shifts by seven bits");
static_assert(SAMPLE_MAX_SLICE<float> / SAMPLE_THREADS + 8 <= 512 && SAMPLE_MAX_SLICE<__nv_bfloat16> / SAMPLE_THREADS + 16 <= 512,
              "a lane's sum of weights, of its share of the vectors and two more, is exact");

// Shared memory of CTA `r` of the cluster, at the place of `p` in this one.
__device__ __forceinline__ unsigned cluster_address(const void* p, int r) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tc_smem(p)), "r"(r));
    return a;
}
__device__ __forceinline__ unsigned cluster_load(const unsigned* p, int r) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_address(p, r)) : "memory");
    return v;
}
__device__ __forceinline__ u64 cluster_load(const u64* p, int r) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_address(p, r)) : "memory");
    return v;
}
__device__ __forceinline__ float cluster_load(const float* p, int r) {
    return __uint_as_float(cluster_load(reinterpret_cast<const unsigned*>(p), r));
}
__device__ __forceinline__ void cluster_store(unsigned* p, int r, unsigned v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_address(p, r)), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_store(u64* p, int r, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_address(p, r)), "l"(v) : "memory");
}

template <class T, int C, bool STAGED>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) k_sample(SampleParams p) {
    constexpr int VE = 16 / sizeof(T);
    extern __shared__ __align__(16) unsigned char smp_raw[];
    T* s_x = reinterpret_cast<T*>(smp_raw);   // STAGED: the slice
    __shared__ SampleShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / C, rank = blockIdx.x % C;
    const auto everywhere = [&]() SAMPLE_INLINE {   // a barrier of all CTAs of the row
        if constexpr (C == 1) __syncthreads();
        else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    };
    const auto read = [&](const auto* ptr, int r) SAMPLE_INLINE {
        if constexpr (C == 1) return *ptr;
        else return cluster_load(ptr, r);
    };
    const auto write = [&](auto* ptr, int r, auto v) SAMPLE_INLINE {
        if constexpr (C == 1) *ptr = v;
        else cluster_store(ptr, r, v);
    };
    // The row starts `shift` elements behind a 16-byte boundary; positions count from that boundary, so that the vectors of
    // a slice are aligned in both memories.  Vectors that reach outside the row are read element by element.
    const T* x = reinterpret_cast<const T*>(p.logits) + (long long)row * p.stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int first = rank * p.slice, vectors = max(0, min(p.slice, p.V + shift - first) + VE - 1) / VE;
    const int per_warp = (vectors + SAMPLE_WARPS - 1) / SAMPLE_WARPS, v0 = min(vectors, warp * per_warp), v1 = min(vectors, v0 + per_warp);
    // what the warp holds in shared memory: its range, later what it moved together (`held` entries); rows that are read again
    // have a ring of copies first, and a list with the entries' places in the warp's range behind it
    T* const mine = STAGED ? s_x + v0 * VE : reinterpret_cast<T*>(smp_raw + SAMPLE_RING_BYTES) + warp * p.list;
    unsigned short* const places =
        reinterpret_cast<unsigned short*>(smp_raw + SAMPLE_RING_BYTES + sizeof(T) * SAMPLE_WARPS * p.list) + warp * p.list;
    unsigned char* const ring = smp_raw + warp * (512 * SAMPLE_RING) + lane * 16;
    bool here = STAGED;
    int held = (v1 - v0) * VE;
    const auto load = [&](int v, T (&e)[VE]) SAMPLE_INLINE {
        const int at = first + v * VE - shift;   // index of the vector's first element in the row
        if (at >= 0 && at + VE <= p.V) {
            *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(x + at);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) e[j] = at + j >= 0 && at + j < p.V ? x[at + j] : T(-INFINITY);
        }
    };

    // A NaN is never drawn; where there are infinite logits they count as zeros and everything else as -infinity.  Rows have
    // neither as a rule: `odd` says whether the warp's range needs the second look.
    bool infinite = false, odd = false;
    const auto clean = [&](T (&e)[VE]) SAMPLE_INLINE {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const float f = to_float(e[j]);
            if (f != f) e[j] = T(-INFINITY);
            else if (infinite) e[j] = f == INFINITY ? T(0.f) : T(-INFINITY);
        }
    };
    // The vectors of the warp's range, 32 at a time: f(v, entries), all lanes together (v past the range: -infinity), as long as
    // it returns true in all of them.
    const auto scan_range = [&](auto&& f) SAMPLE_INLINE {
        alignas(16) T e[VE];
        if constexpr (STAGED) {
            for (int base = v0; base < v1; base += 32) {
                const int v = base + lane;
                if (v < v1) {
                    *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(s_x + v * VE);
                } else {
#pragma unroll
                    for (int j = 0; j < VE; ++j) e[j] = T(-INFINITY);
                }
                if (!f(v, e)) break;
            }
        } else {
            // only the row's first and last vector may reach outside it
            const int in0 = v0 + (first + v0 * VE < shift ? 1 : 0);
            const unsigned in_row = max(0, min(v1, (p.V + shift - first) / VE) - in0);
            const T* from = x + first + (v0 + lane) * VE - shift;
            unsigned slot = 0;
            const auto request = [&](int v, unsigned to) SAMPLE_INLINE {
                if ((unsigned)(v - in0) < in_row)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc_smem(ring) + to), "l"(from) : "memory");
                asm volatile("cp.async.commit_group;" ::: "memory");
                from += 32 * VE;
            };
#pragma unroll
            for (int k = 0; k < SAMPLE_RING - 1; ++k) request(v0 + lane + 32 * k, 512 * k);
            for (int v = v0 + lane; v - lane < v1; v += 32) {
                request(v + 32 * (SAMPLE_RING - 1), (slot + 512 * (SAMPLE_RING - 1)) % (512 * SAMPLE_RING));
                asm volatile("cp.async.wait_group %0;" ::"n"(SAMPLE_RING - 1) : "memory");
                if ((unsigned)(v - in0) < in_row) {
                    *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(ring + slot);
                } else if (v < v1) {
                    load(v, e);
                } else {
#pragma unroll
                    for (int j = 0; j < VE; ++j) e[j] = T(-INFINITY);
                }
                slot = (slot + 512) % (512 * SAMPLE_RING);
                if (odd) clean(e);
                if (!f(v, e)) break;
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
    };

    float top = -INFINITY;
    bool nans = false;
    const auto look = [&](const T (&e)[VE]) SAMPLE_INLINE {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const float f = to_float(e[j]);
            nans |= f != f;
            top = fmaxf(top, f);   // of a number and a NaN: the number
        }
    };
    if constexpr (STAGED) {
#pragma unroll 4
        for (int v = v0 + lane; v < v1; v += 32) {
            alignas(16) T e[VE];
            load(v, e);
            look(e);
            *reinterpret_cast<uint4*>(s_x + v * VE) = *reinterpret_cast<const uint4*>(e);
        }
        if (nans)   // a lane's own vectors
            for (int v = v0 + lane; v < v1; v += 32) clean(*reinterpret_cast<T(*)[VE]>(s_x + v * VE));
    } else {
        scan_range([&](int, const T (&e)[VE]) SAMPLE_INLINE { look(e); return true; });
        odd = __any_sync(0xffffffffu, nans);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if (lane == 0) sh.warp_max[warp] = top;
    if (tid < SAMPLE_TABLE) sh.power[tid] = exp2(-(double)tid / SAMPLE_TABLE);
    for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.count[b] = 0;
    __syncthreads();
    top = sh.warp_max[lane & (SAMPLE_WARPS - 1)];
#pragma unroll
    for (int s = SAMPLE_WARPS / 2; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if constexpr (C > 1) {
        if (tid == 0) sh.top = top;
        everywhere();
#pragma unroll
        for (int r = 0; r < C; ++r) top = fmaxf(top, read(&sh.top, r));
    }

    if (top == -INFINITY) {   // nothing to draw
        if (rank == 0 && tid == 0) p.tokens[row] = p.empty_token;
        everywhere();         // no CTA leaves while another may read its memory
        return;
    }
    if (top == INFINITY) {
        infinite = odd = true;
        top = 0.f;
        if constexpr (STAGED) {
            for (int v = v0 + lane; v < v1; v += 32) clean(*reinterpret_cast<T(*)[VE]>(s_x + v * VE));
            __syncwarp();
        }
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
    // An entry lies t = (top - v) * slope table steps below the largest, n of them to the nearest whole number or next to it:
    // n from FP32 (of entries too far to weigh anything: from SAMPLE_FAR), the rest t - n from FP64.
    const double slope = 1.4426950408889634 * SAMPLE_TABLE / temperature;      // table steps per unit of logit
    const float slope_f = (float)slope, far = SAMPLE_FAR * SAMPLE_TABLE / slope_f;
    const double reach = min_p > 0.0 ? fmax(0.0, -log2(min_p)) * SAMPLE_TABLE : INFINITY;   // table steps that min-p leaves
    const auto steps_below = [&](float v) SAMPLE_INLINE { return ((double)top - (double)v) * slope; };
    const auto whole_steps = [&](float v) SAMPLE_INLINE {
        // a sum with 1.5 * 2^23 is rounded to a whole number
        return __float_as_int(fmaf(fminf(top - v, far), slope_f, 12582912.f)) - __float_as_int(12582912.f);
    };
    const auto weight_at = [&](float v, int n) SAMPLE_INLINE {
        const double whole = __hiloint2double(0x43380000, n) - 6755399441055744.0;   // 1.5 * 2^52 + n, less that
        return fixed_power(n, fma((double)top - (double)v, slope, -whole), sh.power);
    };
    const auto weight_of = [&](float v) SAMPLE_INLINE { return weight_at(v, whole_steps(v)); };
    const auto weight = [&](float v) SAMPLE_INLINE { return (u64)weight_of(v); };
    const auto bin_of = [&](float v) SAMPLE_INLINE { return whole_steps(v) >> SAMPLE_BIN_BITS; };

    float cut = -INFINITY;   // entries under it were dropped
    // Every entry of the warp's range, before anything is moved.
    const auto each_loaded = [&](auto&& f) SAMPLE_INLINE {
        scan_range([&](int, const T (&e)[VE]) {
#pragma unroll
            for (int j = 0; j < VE; ++j) f(to_float(e[j]));
            return true;
        });
    };
    // Every entry that is left.
    const auto each = [&](auto&& f) SAMPLE_INLINE {
        if (here) {
            for (int i = lane; i < held; i += 32) f(to_float(mine[i]));
        } else {
            each_loaded([&](float v) {
                if (v >= cut) f(v);
            });
        }
    };
    const auto block_sum = [&](u64 v) SAMPLE_INLINE {   // over the slice, to total_gt
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
    const auto publish = [&](bool counts, bool masses) SAMPLE_INLINE {
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
    const auto find = [&](u64 carried, auto&& group_sum, auto&& bin_sum, auto&& hit) SAMPLE_INLINE {
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
            if (found >= 0 && lane < C) entries = read(&sh.count[found], lane);
            entries = __reduce_add_sync(0xffffffffu, entries);
            if (lane == 0) {
                sh.bin = found;
                sh.before = before;
                sh.bin_count = entries;
            }
        }
        everywhere();   // found, and no CTA clears what another still reads
    };
    const auto group_counts = [&](int g) SAMPLE_INLINE {
        u64 c = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) c += read(&sh.group_count[g], r);
        return c;
    };
    const auto counts = [&](int b) SAMPLE_INLINE {
        u64 c = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) c += read(&sh.count[b], r);
        return c;
    };
    const auto group_masses = [&](int g) SAMPLE_INLINE {
        u64 m = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) m += read(&sh.group_mass[g], r);
        return m;
    };
    const auto masses = [&](int b) SAMPLE_INLINE {
        u64 m = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) m += read(&sh.mass[b], r);
        return m;
    };
    const auto clear = [&]() SAMPLE_INLINE {
        for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
            sh.count[b] = 0;
            sh.mass[b] = 0;
        }
        __syncthreads();
    };
    // The smallest number that lies in the bins up to `bin`, by a search of the warp over the order of the numbers' bits.
    const auto end_of_bin = [&](int bin) SAMPLE_INLINE {
        unsigned low = order_bits(-3.402823466e38f), high = order_bits(top);
        while (low < high) {
            const unsigned step = (high - low + 31) / 32, at = min(high, low + step * lane);
            const int l = __ffs(__ballot_sync(0xffffffffu, bin_of(from_order_bits(at)) <= bin)) - 1;   // the largest number always is
            if (l < 0) { low = min(high, low + step * 31 + 1); continue; }
            high = min(high, low + step * l);
            low = l == 0 ? high : low + step * (l - 1) + 1;
        }
        return from_order_bits(high);
    };
    // Which entries of a vector are not under the cut.
    const auto in_front = [&](const T (&e)[VE]) SAMPLE_INLINE {
        unsigned stays = 0;
#pragma unroll
        for (int j = 0; j < VE; ++j) stays |= (to_float(e[j]) >= cut ? 1u : 0u) << j;   // a NaN is not
        return stays;
    };
    const auto prefix = [&](int n, int& all) SAMPLE_INLINE {   // over the lanes in front
        int upto = n;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, s);
            if (lane >= s) upto += o;
        }
        all = __shfl_sync(0xffffffffu, upto, 31);
        return upto - n;
    };
    // Walks over the warp's range until more than `most` entries have stayed, which it counts: f(vector, its entries that stay,
    // how many of them are in front of the vector's).
    const auto walk = [&](int most, auto&& f) SAMPLE_INLINE {
        int kept = 0;
        scan_range([&](int v, const T (&e)[VE]) {
            const unsigned stays = in_front(e);
            if (!__any_sync(0xffffffffu, stays)) return true;
            int all;
            const int at = kept + prefix(__popc(stays), all);
            f(v, e, stays, at);
            kept += all;
            __syncwarp();
            return kept <= most;
        });
        return kept;
    };
    // Drops what lies behind `bin`.  Few entries go to the first CTA: true, and sh.mass there holds their keys (ordered by
    // logit, then by place), sh.count their indices.  More move to the front of their warp's range, in order, or into its
    // list.
    unsigned listed = 0;
    const auto keep_up_to = [&](int bin) SAMPLE_INLINE {
        cut = end_of_bin(bin);
        int n = 0;
        if constexpr (STAGED) {
            scan_range([&](int, const T (&e)[VE]) { n += __popc(in_front(e)); return true; });
            n = __reduce_add_sync(0xffffffffu, n);
        } else {
            n = walk(p.list, [&](int v, const T (&e)[VE], unsigned stays, int at) {
#pragma unroll
                for (int j = 0; j < VE; ++j)
                    if (stays >> j & 1) {
                        if (at < p.list) {
                            places[at] = (unsigned short)((v - v0) * VE + j);
                            mine[at] = e[j];
                        }
                        ++at;
                    }
            });
            here = n <= p.list;   // else the range stays where it is, and there are more than go to the first CTA
            held = n;
        }
        if (lane == 0) sh.warp_eq[warp] = n;
        __syncthreads();
        unsigned in_warps = lane < SAMPLE_WARPS ? sh.warp_eq[lane] : 0;
        const unsigned before_warp = __reduce_add_sync(0xffffffffu, lane < warp ? in_warps : 0);
        in_warps = __reduce_add_sync(0xffffffffu, in_warps);
        if (tid == 0) sh.kept = in_warps;
        everywhere();
        const unsigned in_slices = lane < C ? read(&sh.kept, lane) : 0;
        const unsigned before_slice = __reduce_add_sync(0xffffffffu, lane < rank ? in_slices : 0);
        listed = __reduce_add_sync(0xffffffffu, in_slices);
        const bool few = listed <= SAMPLE_THREADS;
        const auto list = [&](unsigned place, float v, int index) SAMPLE_INLINE {
            write(&sh.mass[place], 0, (u64)order_bits(v) << 32 | (0xffffffffu - place));
            write(&sh.count[place], 0, (unsigned)index);
        };
        if constexpr (STAGED) {
            held = walk(n, [&](int v, const T (&e)[VE], unsigned stays, int at) {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < VE; ++j)
                    if (stays >> j & 1) {
                        if (few) list(before_slice + before_warp + at, to_float(e[j]), first + v * VE + j - shift);
                        else mine[at] = e[j];   // never ahead of what the warp has read
                        ++at;
                    }
            });
        } else if (few) {   // 512 at most: they are in the lists
            for (int i = lane; i < held; i += 32)
                list(before_slice + before_warp + i, to_float(mine[i]), first + v0 * VE + places[i] - shift);
        }
        if (few) everywhere();
        return few;
    };
    const auto block_scan = [&](u64 v, u64& all) SAMPLE_INLINE {   // sum of the threads up to this one, and of all
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
    const auto uniform_part = [&](u64 all) SAMPLE_INLINE {   // the whole part of u times the sum
        const float u = p.uniform[row];
        const double clipped = u > 0.f ? fmin((double)u, 1.0 - 0x1p-53) : 0.0;   // a NaN counts as zero
        return __umul64hi(all, (u64)(clipped * 0x1p64));
    };
    // The first `n` threads' keys in descending order, zeros behind, through `scratch`.  Every key is compared with every other
    // one, by as many threads as there are for it: two barriers where a sorting network takes two for every step between
    // warps (132 keys: 9000 clocks in one).
    const auto sort_down = [&](auto key, unsigned n, auto* scratch) SAMPLE_INLINE {
        __syncthreads();
        if (tid < n) scratch[tid] = key;
        __syncthreads();
        const int parts_log2 = min(5, 31 - __clz((int)(SAMPLE_THREADS / n))), parts = 1 << parts_log2;
        const unsigned i = (unsigned)tid >> parts_log2;
        decltype(key) mine_of = 0;
        unsigned above = 0;
        if (i < n) {
            mine_of = scratch[i];
#pragma unroll 4
            for (unsigned j = tid & (parts - 1); j < n; j += parts) {
                const auto other = scratch[j];
                above += other > mine_of || (other == mine_of && j < i) ? 1u : 0u;
            }
        }
        for (int s = 1; s < parts; s <<= 1) above += __shfl_xor_sync(0xffffffffu, above, s);
        __syncthreads();
        if (i < n && (tid & (parts - 1)) == 0) scratch[above] = mine_of;
        __syncthreads();
        key = tid < n ? scratch[tid] : 0;
        return key;
    };
    // The rest of the row's work where few candidates are left, by the first CTA: one a thread, sorted by logit and place.
    const auto draw_from_list = [&](unsigned k, bool by_p, double target, bool sum_first) SAMPLE_INLINE {
        if (rank != 0) return;
        u64 key = tid < (int)listed ? sh.mass[tid] : 0ull;
        if (k < listed || by_p) key = sort_down(key, listed, sh.mass);
        const unsigned place = 0xffffffffu - (unsigned)key;
        const float v = from_order_bits((unsigned)(key >> 32));
        const u64 w = tid < (int)listed && tid < (int)k ? weight(v) : 0ull;
        bool stays = w != 0 && steps_below(v) <= reach;
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
    unsigned ties = 0;
    // what refine() leaves for the draw: the lane's sum of the weights in front of the border's step, and the step's entries in
    // the warp's range where it is read again (-1: not all of them fitted into the list)
    double front = 0.0;
    bool fronted = false;
    int stepped = -1;

    const auto each_in_step = [&](auto&& f) SAMPLE_INLINE {   // of the step at least: in the list, where that holds it
        if (!here && stepped < 0) {
            each_loaded(f);
            return;
        }
        const int n = here ? held : stepped;
        for (int i = lane; i < n; i += 32) f(to_float(mine[i]));
    };
    // The border inside the bin `step`, on the edge of what a running sum reaches: of weights, `target`; of counts, `count`.
    // `before` is that sum over the bins in front; with `sum_front` it is added up here.
    // False: the border is in front of the step.
    const auto refine = [&](int step, bool by_mass, unsigned count, double target, u64 before, bool sum_front) SAMPLE_INLINE {
        unsigned n = 0;
        front = 0.0;
        fronted = !STAGED && sum_front;   // of a row in shared memory the saving is lost on registers (32000 logits: 10.2 us, 9.9)
        if (STAGED || here) {
            for (int i = lane; i < held; i += 32) {
                const float v = to_float(mine[i]);
                const int b = bin_of(v);
                if (b == step) n += v > -INFINITY && !(v < edge);
                else if (sum_front && b < step) front += weight_of(v);
            }
            n = __reduce_add_sync(0xffffffffu, n);
        } else {   // nothing under the cut is in the step or in front of it
            scan_range([&](int, const T (&e)[VE]) {
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const float v = to_float(e[j]);
                    const int b = bin_of(v);
                    const bool in = b == step && v > -INFINITY && !(v < edge);
                    if (sum_front && b < step) front += weight_of(v);
                    const unsigned lanes = __ballot_sync(0xffffffffu, in);
                    const unsigned at = n + __popc(lanes & ((1u << lane) - 1));
                    if (in && at < p.list) mine[at] = e[j];
                    n += __popc(lanes);
                }
                return true;
            });
            stepped = n <= p.list ? (int)n : -1;
        }
        if (lane == 0) sh.warp_eq[warp] = n;
        if (sum_front) block_sum((u64)front);
        else __syncthreads();
        unsigned in_warps = lane < SAMPLE_WARPS ? sh.warp_eq[lane] : 0;
        const unsigned before_warp = __reduce_add_sync(0xffffffffu, lane < warp ? in_warps : 0);
        in_warps = __reduce_add_sync(0xffffffffu, in_warps);
        if (tid == 0) sh.in_step = in_warps;
        everywhere();
        const unsigned in_slices = lane < C ? read(&sh.in_step, lane) : 0;
        const unsigned before_slice = __reduce_add_sync(0xffffffffu, lane < rank ? in_slices : 0);
        const unsigned all = __reduce_add_sync(0xffffffffu, in_slices);
        if (sum_front)
            for (int r = 0; r < C; ++r) before += read(&sh.total_gt, r);
        if (sum_front && !((double)before < target)) {
            everywhere();   // in_step and total_gt have been read
            return false;
        }
        if (all <= SAMPLE_THREADS) {
            // every CTA gets all entries of the step and sorts them (they are in the lists: a warp's takes more than 512)
            unsigned at = before_slice + before_warp;
            const int on_hand = here ? held : stepped;
            for (int i0 = 0; i0 < on_hand; i0 += 32) {
                const float v = i0 + lane < on_hand ? to_float(mine[i0 + lane]) : -INFINITY;
                const bool in = v > -INFINITY && !(v < edge) && bin_of(v) == step;
                const unsigned lanes = __ballot_sync(0xffffffffu, in);
                if (in)
                    for (int r = 0; r < C; ++r) write(&sh.count[at + __popc(lanes & ((1u << lane) - 1))], r, order_bits(v));
                at += __popc(lanes);
            }
            everywhere();
            const unsigned key = sort_down(tid < all ? sh.count[tid] : 0u, all, sh.count);
            bool is_it = by_mass ? false : tid == count - 1 - (unsigned)before;
            if (by_mass) {
                const u64 w = tid < all ? weight(from_order_bits(key)) : 0ull;
                u64 sum;
                const u64 upto = before + block_scan(w, sum);
                is_it = (double)(upto - w) < target && !((double)upto < target);
            }
            if (is_it) {
                sh.edge = from_order_bits(key);
                sh.ties = tid;
            }
            __syncthreads();
            edge = sh.edge;
            ties = __syncthreads_count(tid <= sh.ties && from_order_bits(key) == edge && tid < all);
            everywhere();   // sh.count may be used again
            return true;
        }
        unsigned low = 0xffffffffu, high = 0;
        each_in_step([&](float v) {
            if (bin_of(v) != step || !(v > -INFINITY) || v < edge) return;
            const unsigned k = order_bits(v);
            low = min(low, k);
            high = max(high, k);
        });
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        if (tid == 0) {
            sh.low = 0xffffffffu;
            sh.high = 0;
            sh.bin_count = all;
            sh.before = before;
        }
        __syncthreads();
        if (lane == 0) {
            atomicMin(&sh.low, low);
            atomicMax(&sh.high, high);
        }
        everywhere();
#pragma unroll
        for (int r = 0; r < C; ++r) {
            low = min(low, read(&sh.low, r));
            high = max(high, read(&sh.high, r));
        }
        while (low != high) {
            const int width = 32 - __clz(high - low), down = width > 10 ? width - 10 : 0;   // 1024 bins
            const u64 carried = sh.before;
            clear();
            each_in_step([&](float v) {
                const unsigned k = order_bits(v);
                if (k < low || k > high) return;
                const int b = (int)((high - k) >> down);
                if (by_mass) atomicAdd(&sh.mass[b], weight(v));
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
        ties = count - (unsigned)sh.before;
        if (by_mass) {
            const u64 w = weight(edge), in_front_of = sh.before;
            const unsigned equal = sh.bin_count;
            ties = (unsigned)fmin(fmax(ceil((target - (double)in_front_of) / (double)w), 1.0), (double)equal);
            while (ties > 1 && !((double)(in_front_of + (ties - 1) * w) < target)) --ties;
            while (ties < equal && (double)(in_front_of + ties * w) < target) ++ties;
        }
        everywhere();   // sh.before and sh.bin_count are read by everyone before they change
        return true;
    };

    const int min_p_bin = reach < SAMPLE_RANGE * SAMPLE_TABLE ? ((int)reach >> SAMPLE_BIN_BITS) + 1 : SAMPLE_BINS;
    const bool by_k = top_k > 1 && top_k < p.V, by_p = top_k != 1 && top_p < 1.0;
    double target = 0.0;
    // the borders still to be found: of top-k, of top-p at the end of what is left, of top-p anywhere in what is left
    enum { DONE, TOP_K, TOP_P, TOP_P_LEFT };
    if (top_k == 1) {
        // the first entry that equals the largest
        unsigned at = 0xffffffffu;
        scan_range([&](int v, const T (&e)[VE]) {
#pragma unroll
            for (int j = VE - 1; j >= 0; --j)
                if (to_float(e[j]) == top) at = min(at, (unsigned)(first + v * VE + j - shift));
            return true;
        });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) sh.warp_eq[warp] = at;
        __syncthreads();
        if (warp == 0) {
            at = __reduce_min_sync(0xffffffffu, sh.warp_eq[lane & (SAMPLE_WARPS - 1)]);
            if (lane == 0) sh.low = at;
        }
        everywhere();
        if (rank == 0 && warp == 0) {
            at = __reduce_min_sync(0xffffffffu, read(&sh.low, lane & (C - 1)));
            if (lane == 0) p.tokens[row] = at;
        }
        everywhere();   // no CTA leaves while another may read its memory
        return;
    }
    int step = 0, keep = SAMPLE_BINS;   // the step of the first rule's border, and the last bin that is kept
    int rule = DONE;
    if (by_k) {
        each_loaded([&](float v) {
            if (v > -INFINITY) atomicAdd(&sh.count[bin_of(v)], 1u);
        });
        publish(true, false);
        find(0, group_counts, counts, [&](u64 a, u64 b) { return a < (unsigned)top_k && b >= (unsigned)top_k; });
        step = sh.bin;   // -1: fewer candidates than top-k keeps
        keep = step < 0 ? SAMPLE_BINS - 1 : step;
        if (!by_p && min_p_bin < keep) keep = min_p_bin;   // all that is in front of that is among the first k
        else if (step >= 0) rule = TOP_K;
        if (by_p && rule == DONE) rule = TOP_P_LEFT;
    } else if (by_p) {
        // the sum of all weights, and a histogram of their upper bits (against 2^(43 - a), the binade of the bin), as many as leave a
        // counter of 32 bits room for a slice of equal logits: its running sums are not above the true ones, so the border is
        // not behind the bin in which they reach the target
        constexpr int PER_BINADE = SAMPLE_TABLE >> SAMPLE_BIN_BITS;
        constexpr int BITS = SAMPLE_BIN_WEIGHT_BITS<T, STAGED>;
        static_assert(SAMPLE_COUNTERS_HOLD<T, STAGED>, "histogram of weights");
        double sum = 0.0;
        each_loaded([&](float v) {
            const int n = whole_steps(v);
            const double w = weight_at(v, n);
            sum += w;
            const int high = __double2hiint(w), binades = (high >> 20) - (1023 + 43) + (n >> 7);   // over 2^(43 - a): 0, or 1 at its end
            if (high != 0) atomicAdd(&sh.count[n >> SAMPLE_BIN_BITS], (unsigned)((high & 0xfffff) | 0x100000) << (binades + 1) >> (22 - BITS));
        });
        block_sum((u64)sum);
        for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
            const int up = SAMPLE_WEIGHT_BITS - BITS - b / PER_BINADE;
            sh.mass[b] = up >= 0 ? (u64)sh.count[b] << up : (u64)sh.count[b] >> -up;
        }
        publish(false, true);
        u64 all = 0;
        for (int r = 0; r < C; ++r) all += read(&sh.total_gt, r);
        target = top_p * (double)all;
        find(0, group_masses, masses, [&](u64 a, u64 b) { return (double)a < target && !((double)b < target); });
        step = sh.bin < 0 ? SAMPLE_BINS - 1 : sh.bin;
        keep = min(step, min_p_bin);
        if (step <= min_p_bin) rule = TOP_P;
    } else {
        keep = min_p_bin;
    }
    const u64 in_front_of_step = sh.before;
    if (keep < SAMPLE_BINS && keep_up_to(keep)) {
        draw_from_list(by_k ? (unsigned)top_k : SAMPLE_THREADS, by_p, target, by_k);
        return;
    }
    if (by_p && !by_k && step > min_p_bin) {
        // min-p cuts in front of the last step in which top-p's border can lie.  The border is behind all that is left if the first
        // step in which it can lie is: of a weight the histogram lost less than its 2^-(BITS - 1), 2^-13 at most, of a bin
        // of a slice less than one (8192 in all)
        const double least = target * (1.0 - 0x1p-13) - 0x1p14;
        find(0, group_masses, masses, [&](u64, u64 b) { return !((double)b < least); });
        if (sh.bin >= 0 && sh.bin <= min_p_bin) rule = TOP_P_LEFT;
    }
    while (rule != DONE) {
        if (rule == TOP_P_LEFT) {
            if (by_k) {   // the weight of what top-k keeps
                double sum = 0.0;
                each([&](float v) { if (v > edge) sum += weight_of(v); });
                block_sum((u64)sum);
                everywhere();
                u64 all = edge > -INFINITY ? ties * weight(edge) : 0ull;
                for (int r = 0; r < C; ++r) all += read(&sh.total_gt, r);
                target = top_p * (double)all;
            }
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
            step = sh.bin;
            if (step < 0) break;   // min-p cut in front of the border
        }
        const bool found = refine(step, rule != TOP_K, (unsigned)top_k, target, rule == TOP_K ? in_front_of_step : rule == TOP_P ? 0 : sh.before,
                                  rule == TOP_P);
        rule = rule == TOP_K && by_p ? TOP_P_LEFT : rule == TOP_P && !found ? TOP_P_LEFT : DONE;
    }

    // the draw
    const auto drawn_weight = [&](float v) SAMPLE_INLINE -> u64 {
        return reach == INFINITY || steps_below(v) <= reach ? weight(v) : 0ull;
    };
    const u64 edge_weight = edge > -INFINITY ? drawn_weight(edge) : 0ull;
    double gt_sum = 0.0;
    unsigned eq = 0;
    if (cut == -INFINITY) {   // no rule: no border either
        each_loaded([&](float v) { gt_sum += weight_of(v); });
    } else if (fronted && reach == INFINITY) {
        // every entry in front of the step stays, none behind it
        if (!here && stepped >= 0) {
            for (int i = lane; i < stepped; i += 32) {
                const float v = to_float(mine[i]);
                if (v > edge) gt_sum += weight_of(v);
                else if (v == edge) ++eq;
            }
        } else {
            each([&](float v) {
                if (v == edge) ++eq;
                else if (v > edge && bin_of(v) == step) gt_sum += weight_of(v);
            });
        }
    } else {
        front = 0.0;
        each([&](float v) {
            if (v > edge) gt_sum += reach == INFINITY || steps_below(v) <= reach ? weight_of(v) : 0.0;
            else if (v == edge) ++eq;
        });
    }
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) sh.warp_eq[warp] = eq;
    block_sum((u64)front + (u64)gt_sum);
    if (tid == 0) {
        unsigned b = 0;
        for (int w = 0; w < SAMPLE_WARPS; ++w) b += sh.warp_eq[w];
        sh.total_eq = b;
    }
    everywhere();
    u64 all = 0, before = 0, own = 0;
    unsigned seen = 0, passed = 0;   // candidates on the edge before this slice, then before this warp
    for (int r = 0; r < C; ++r) {
        const unsigned e = read(&sh.total_eq, r), keep = passed < ties ? min(e, ties - passed) : 0;
        const u64 sum = read(&sh.total_gt, r) + keep * edge_weight;
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
    if (!here) {   // over the range itself, a vector a lane
        scan_range([&](int v, const T (&e)[VE]) {
            u64 sum = 0;
            int on = 0;
            const unsigned stays = in_front(e);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float f = to_float(e[j]);
                if (!(stays >> j & 1)) continue;
                if (f > edge) sum += drawn_weight(f);
                else if (f == edge && f > -INFINITY) ++on;
            }
            int on_all;
            const unsigned ahead = seen + prefix(on, on_all);
            sum += (ahead < ties ? min((unsigned)on, ties - ahead) : 0) * edge_weight;
            u64 upto = sum;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const u64 o = __shfl_up_sync(0xffffffffu, upto, s);
                if (lane >= s) upto += o;
            }
            const u64 from = before + upto - sum;
            if (drawn >= from && drawn < from + sum) {
                u64 run = from;
                unsigned k = ahead;
                for (int j = 0; j < VE; ++j) {
                    const float f = to_float(e[j]);
                    if (!(stays >> j & 1)) continue;
                    if (f > edge) run += drawn_weight(f);
                    else if (f == edge && f > -INFINITY && k++ < ties) run += edge_weight;
                    if (run > drawn) {
                        p.tokens[row] = first + v * VE + j - shift;
                        break;
                    }
                }
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
            seen += on_all;
            return drawn >= before;
        });
        return;
    }
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
    if (!STAGED) place = places[place];
    if (!STAGED || cut == -INFINITY) {
        if (lane == 0) p.tokens[row] = first + v0 * VE + place - shift;
        return;
    }
    // the place-th of those entries of the warp's range that were kept, counted again in the row itself
    constexpr int AHEAD = 4;
    for (int base = v0; base < v1; base += 32 * AHEAD) {
        alignas(16) T e[AHEAD][VE];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (base + 32 * a + lane < v1) {
                load(base + 32 * a + lane, e[a]);
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j) e[a][j] = T(-INFINITY);
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            clean(e[a]);
            const unsigned stays = in_front(e[a]);
            int all_kept;
            const int n = __popc(stays), from = prefix(n, all_kept);
            if (place >= from && place < from + n)
                for (int j = 0, k = from; j < VE; ++j)
                    if (stays >> j & 1 && k++ == place) p.tokens[row] = first + (base + 32 * a + lane) * VE + j - shift;
            if (place < all_kept) return;
            place -= all_kept;
        }
    }
}

#undef SAMPLE_INLINE

}  // namespace sd
