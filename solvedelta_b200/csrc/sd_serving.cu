// C ABI of the serving operators: 8-bit projections and token sampling (declarations: include/solvedelta_b200.h).
#include "../../include/solvedelta_b200.h"
#include "sd_int8.cuh"
#include "sd_internal.h"
#include "sd_sampling.cuh"

namespace {

using namespace sd;

bool aligned(const void* p, size_t n = 16) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int status_of(cudaError_t e) {
    const cudaError_t last = cudaGetLastError();
    return e == cudaSuccess && last == cudaSuccess ? SD_OK : SD_ERR_LAUNCH_FAILED;
}

// Opt-in to dynamic shared memory above the default, once per device and kernel, always to the same size.
template <auto KERNEL>
cudaError_t allow_smem(size_t most) {
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev])) return e;
    if ((e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most)) != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) done[dev] = true;
    return cudaSuccess;
}
// `chained`: the kernel may start while the one before it in the stream still runs (it waits for it itself).
template <auto KERNEL, class... Args>
int launch(unsigned grid, unsigned threads, size_t smem, size_t most_smem, int cluster, bool chained, cudaStream_t stream, const Args&... args) {
    if (most_smem > 0) {
        const cudaError_t e = allow_smem<KERNEL>(most_smem);
        if (e != cudaSuccess) return SD_ERR_NO_DEVICE;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2] = {};
    int n = 0;
    if (chained) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = cluster;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    return status_of(cudaLaunchKernelEx(&cfg, KERNEL, args...));
}

constexpr int MAX_K = 131072;   // 127 * 127 * K stays below 2^31
int padded(int K) { return (K + 15) / 16 * 16; }

// ---- quantised rows ----
template <class T, bool VEC, int W, int H>
int quantize_launch(const QuantizeParams& p, bool chained, cudaStream_t stream) {
    return launch<k_quantize_rows<T, VEC, W, H>>((unsigned)((p.rows * W + 7) / 8), QUANT_THREADS, 0, 0, 1, chained, stream, p);
}
template <class T, bool VEC, int H>
int quantize_width(const QuantizeParams& p, bool chained, cudaStream_t stream) {
    // as few warps a row as hold it in registers (16384 x 2048: 28 us with one, 38 with eight), but more while the SMs are not full
    // of warps (64 x 1024: 1.9 us with eight, 2.9 with one)
    const auto enough = [&](int w) { return (long long)w * 256 * H >= p.K && p.rows * w >= 148 * 16; };
    if (enough(1)) return quantize_launch<T, VEC, 1, H>(p, chained, stream);
    if (enough(2)) return quantize_launch<T, VEC, 2, H>(p, chained, stream);
    if (enough(4)) return quantize_launch<T, VEC, 4, H>(p, chained, stream);
    if (p.K <= 8 * 256) return quantize_launch<T, VEC, 8, 1>(p, chained, stream);
    return quantize_launch<T, VEC, 8, H>(p, chained, stream);
}
int quantize(const sd_quantize_rows_args* a, bool chained, cudaStream_t stream) {
    QuantizeParams p{};
    p.rows = a->rows; p.K = a->K;
    p.x = a->x; p.x_stride = a->x_stride;
    p.q = reinterpret_cast<signed char*>(a->q); p.q_stride = a->q_stride;
    p.scale = a->scale;
    const bool f32 = a->x_type == SD_F32;
    const bool vec = aligned(a->x) && a->x_stride % (f32 ? 4 : 8) == 0 && a->K % 8 == 0;
    if (f32) return vec ? quantize_width<float, true, 4>(p, chained, stream) : quantize_width<float, false, 4>(p, chained, stream);
    return vec ? quantize_width<__nv_bfloat16, true, 8>(p, chained, stream) : quantize_width<__nv_bfloat16, false, 8>(p, chained, stream);
}

// ---- products ----
// Tensor map of int8 rows [rows][K]: boxes of `box_rows` rows by 128 bytes, 128-byte swizzle.
bool int8_map(CUtensorMap* map, const void* base, long long rows, int K, long long stride, int box_rows) {
    const TensorMapEncodeFn encode = map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)I8_BK, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool GATED, bool F32, bool PAIR>
int launch_matmul(Int8Params p, const sd_int8_linear_args* a, const void* q, long long q_stride, bool chained, cudaStream_t stream) {
    constexpr int OUTS = GATED ? BN / 2 : BN, CTAS = PAIR ? 2 : 1;
    CUtensorMap x_map, w_map;
    int* fault = fault_word();
    if (fault == nullptr) return SD_ERR_NO_DEVICE;
    if (!int8_map(&x_map, q, p.M, p.K, q_stride, I8_BM) || !int8_map(&w_map, a->weight, a->N, p.K, a->weight_stride, PAIR || GATED ? BN / 2 : BN))
        return SD_ERR_LAUNCH_FAILED;
    p.tiles_m = (p.M + CTAS * I8_BM - 1) / (CTAS * I8_BM);
    p.tiles_n = (p.outs + OUTS - 1) / OUTS;
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    if (tiles > 0x7fffffffLL - 148) return SD_ERR_UNSUPPORTED_SHAPE;
    const unsigned workers = (unsigned)(tiles < 148 / CTAS ? tiles : 148 / CTAS);
    return launch<k_int8_matmul<BN, GATED, F32, PAIR>>(workers * CTAS, I8_THREADS, Int8Tile<BN, PAIR>::SMEM, Int8Tile<BN, PAIR>::SMEM, CTAS,
                                                       chained, stream, p, x_map, w_map, fault);
}
// How many CTAs share a tile of 128 x 64 (as a power of two): as many as the SMs have room for, four steps of K each at least
// (64 x 5632 x 2048: 8.7 us with four, 16.2 with one; 128 x 2816 x 1024: 7.5 and 9.9).
int split_log2(long long tiles, int K) {
    const int blocks = (K + I8_BK - 1) / I8_BK;
    int n = 0;
    while (n < 3 && (tiles << (n + 1)) <= 148 && blocks >> (n + 1) >= 4) ++n;
    return n;
}
template <bool GATED, bool F32>
int launch_split(Int8Params p, const sd_int8_linear_args* a, const void* q, long long q_stride, int ctas_log2, bool chained, cudaStream_t stream) {
    using Tile = Int8Tile<I8_SPLIT_BN, false>;
    constexpr int OUTS = GATED ? I8_SPLIT_BN / 2 : I8_SPLIT_BN;
    CUtensorMap x_map, w_map;
    int* fault = fault_word();
    if (fault == nullptr) return SD_ERR_NO_DEVICE;
    if (!int8_map(&x_map, q, p.M, p.K, q_stride, I8_BM) || !int8_map(&w_map, a->weight, a->N, p.K, a->weight_stride, OUTS)) return SD_ERR_LAUNCH_FAILED;
    p.tiles_m = (p.M + I8_BM - 1) / I8_BM;
    p.tiles_n = (p.outs + OUTS - 1) / OUTS;
    const int blocks = (p.K + I8_BK - 1) / I8_BK, ctas = 1 << ctas_log2, per = (blocks + ctas - 1) / ctas;
    return launch<k_int8_split<GATED, F32>>((unsigned)(p.tiles_m * p.tiles_n * ctas), I8_THREADS, Tile::SMEM, Tile::SMEM, ctas, chained, stream, p,
                                            ctas_log2, per, x_map, w_map, fault);
}
template <bool GATED, bool F32>
int matmul_tile(const Int8Params& p, const sd_int8_linear_args* a, const void* q, long long q_stride, bool chained, cudaStream_t stream) {
    const auto tiles = [&](int bm, int bn) {
        const int outs = GATED ? bn / 2 : bn;
        return (long long)((p.M + bm - 1) / bm) * ((p.outs + outs - 1) / outs);
    };
    // Pairs of CTAs from half of the SMs on (700 x 2048 x 4096, 48 tiles: 11.3 us, tiles of one CTA 14.9; 300 x 2048 x 2048, 16
    // tiles: 10.9 against 8.5); else the wider tile while it gives every SM one (2048 x 1024 x 2816: 128 columns 13.5 us, 64 18.2;
    // 128 x 1024 x 5632, 44 tiles of 128 columns: 6.4 against 5.9).  Just under that bound the narrow tiles take a second round
    // that is nearly empty (64 x 2048 x 11264 with SwiGLU, 88 tiles of 128 columns or 176 of 64: 13.5 us, 3.6 for its bytes).
    if (tiles(256, 256) >= 37 && p.M > 128) return launch_matmul<256, GATED, F32, true>(p, a, q, q_stride, chained, stream);
    if (tiles(128, 128) >= 148) return launch_matmul<128, GATED, F32, false>(p, a, q, q_stride, chained, stream);
    const int ctas_log2 = split_log2(tiles(128, 64), p.K);
    if (ctas_log2 > 0) return launch_split<GATED, F32>(p, a, q, q_stride, ctas_log2, chained, stream);
    return launch_matmul<64, GATED, F32, false>(p, a, q, q_stride, chained, stream);
}
int matmul(const Int8Params& p, const sd_int8_linear_args* a, const void* q, long long q_stride, bool chained, cudaStream_t stream) {
    if (a->swiglu) return p.out_f32 ? matmul_tile<true, true>(p, a, q, q_stride, chained, stream)
                                    : matmul_tile<true, false>(p, a, q, q_stride, chained, stream);
    return p.out_f32 ? matmul_tile<false, true>(p, a, q, q_stride, chained, stream)
                     : matmul_tile<false, false>(p, a, q, q_stride, chained, stream);
}

size_t token_smem(int M, int K) { return (size_t)(M * int8_pitch(K)); }
template <int RG, int CG, bool GATED, class T>
int launch_token(const Int8TokenParams& p, bool chained, cudaStream_t stream) {
    constexpr int WIDTH = GATED ? 8 : 8 * CG;
    const int tiles = (p.o.outs + WIDTH - 1) / WIDTH;
    const size_t smem = token_smem(p.o.M, p.o.K);
    const int resident = 148 * (smem <= 96 * 1024 ? 2 : 1);
    return launch<k_int8_token<RG, CG, GATED, T>>((unsigned)(tiles < resident ? tiles : resident), 256, smem, I8_TOKEN_SMEM, 1,
                                                       chained, stream, p);
}
template <int RG, class T>
int token_width(const Int8TokenParams& p, bool gated, bool chained, cudaStream_t stream) {
    if (gated) return launch_token<RG, 2, true, T>(p, chained, stream);
    // 16 columns a tile while that keeps most SMs busy (one row, 1024 x 2048: 2.9 us, with 8 columns 3.1; 2048 x 4096: 4.3 and 4.8),
    // else 8 (2816 x 1024: 3.2 us, with 16 columns 3.7)
    return p.o.outs >= 16 * 128 ? launch_token<RG, 2, false, T>(p, chained, stream)
                                : launch_token<RG, 1, false, T>(p, chained, stream);
}
template <class T>
int token_rows(const Int8TokenParams& p, bool gated, bool chained, cudaStream_t stream) {
    if (p.o.M <= 8) return token_width<1, T>(p, gated, chained, stream);
    return token_width<2, T>(p, gated, chained, stream);
}
bool token_takes(const sd_int8_linear_args* a) { return a->rows <= I8_TOKEN_ROWS && token_smem((int)a->rows, a->K) <= I8_TOKEN_SMEM; }
// Few entries: every CTA quantises the rows for itself, which saves a launch; past that it costs more (4 x 1024 entries: 5.9 us
// against 6.0, 8 x 1024: 7.9 against 6.2).
constexpr long long TOKEN_FUSED_ENTRIES = 4096;
bool token_fuses(const sd_int8_linear_args* a) {
    return token_takes(a) && a->x_type == SD_BF16 && aligned(a->x) && a->x_stride % 8 == 0 && a->K % 8 == 0 && a->rows * a->K <= TOKEN_FUSED_ENTRIES;
}

size_t q_bytes(const sd_int8_linear_args* a) { return ((size_t)a->rows * padded(a->K) + 255) / 256 * 256; }

// ---- sampling ----
constexpr size_t SAMPLE_LIST_BYTES = 60 * 1024;
constexpr long long SAMPLE_L2 = 96 << 20;       // of 126 MB
static_assert(2 * (SAMPLE_STAGED + sizeof(SampleShared) + 1024) <= 228 * 1024 &&
              2 * (SAMPLE_RING_BYTES + SAMPLE_LIST_BYTES + sizeof(SampleShared) + 1024) <= 228 * 1024, "two CTAs an SM");
template <class T, int C>
int launch_sample(SampleParams p, long long rows, cudaStream_t stream) {
    constexpr int VE = 16 / sizeof(T);
    // rows may start up to VE - 1 elements behind a 16-byte boundary
    p.slice = ((p.V + VE - 1 + C - 1) / C + VE - 1) / VE * VE;
    const size_t bytes = (size_t)p.slice * sizeof(T);
    if (bytes <= SAMPLE_STAGED)
        return launch<k_sample<T, C, true>>((unsigned)(rows * C), SAMPLE_THREADS, bytes, SAMPLE_STAGED, C, false, stream, p);
    constexpr int list = SAMPLE_LIST_BYTES / SAMPLE_WARPS / (sizeof(T) + sizeof(unsigned short));
    static_assert(list > SAMPLE_THREADS, "what the CTAs sort fits into one warp's list");
    p.list = list;
    constexpr size_t smem = SAMPLE_RING_BYTES + SAMPLE_LIST_BYTES;
    return launch<k_sample<T, C, false>>((unsigned)(rows * C), SAMPLE_THREADS, smem, smem, C, false, stream, p);
}
template <class T>
int sample(const SampleParams& p, long long rows, cudaStream_t stream) {
    // as many CTAs a row as the SMs take at once, two on each, with 2048 entries at least; and so many that the rows in work
    // at a time, which are read three times, stay in L2 (512 rows of 128000 in FP32, top-p 0.95, logits N(0, 4): 618 us with one
    // CTA a row, 563 with two, 648 with four; N(0, 16): 277, 280, 354)
    const auto worth = [&](int c) {
        return p.V >= c * 2048 && (rows * c <= 2 * 148 || 2 * 148 / (c / 2) * (long long)p.V * (int)sizeof(T) > SAMPLE_L2);
    };
    // by the second condition no part of a row is longer than this
    static_assert(SAMPLE_L2 / (2 * 148 * (int)sizeof(T)) + 16 <= SAMPLE_MAX_SLICE<T>, "longest slices");
    if (worth(8)) return launch_sample<T, 8>(p, rows, stream);
    if (worth(4)) return launch_sample<T, 4>(p, rows, stream);
    if (worth(2)) return launch_sample<T, 2>(p, rows, stream);
    return launch_sample<T, 1>(p, rows, stream);
}

}  // namespace

extern "C" {

int sd_quantize_rows(const sd_quantize_rows_args* a, void* stream_) {
    if (!a || a->rows <= 0 || a->K <= 0 || !a->x || !a->q || !a->scale || (a->x_type != SD_BF16 && a->x_type != SD_F32))
        return SD_ERR_INVALID_ARGUMENT;
    if (a->q_stride < padded(a->K) || a->q_stride % 16 != 0 || !aligned(a->q)) return SD_ERR_INVALID_ARGUMENT;
    if (a->rows > 0x7fffffffLL || a->K > MAX_K) return SD_ERR_UNSUPPORTED_SHAPE;
    return quantize(a, false, reinterpret_cast<cudaStream_t>(stream_));
}

size_t sd_int8_linear_scratch_bytes(const sd_int8_linear_args* a) {
    if (!a || a->rows <= 0 || a->K <= 0 || a->x_type == SD_I8 || token_fuses(a)) return 0;
    return q_bytes(a) + (size_t)a->rows * 4;
}

int sd_int8_linear(const sd_int8_linear_args* a, void* stream_) {
    if (!a || a->rows <= 0 || a->N <= 0 || a->K <= 0 || !a->x || !a->weight || !a->weight_scale || !a->y ||
        (a->swiglu && a->N % 2 != 0) || (a->y_type != SD_BF16 && a->y_type != SD_F32) || a->x_type < SD_BF16 || a->x_type > SD_I8 ||
        (a->x_type == SD_I8 && !a->x_scale) || (a->bias && a->bias_type != SD_BF16 && a->bias_type != SD_F32))
        return SD_ERR_INVALID_ARGUMENT;
    if (!aligned(a->weight) || a->weight_stride % 16 != 0 || a->weight_stride < padded(a->K) ||
        (a->x_type == SD_I8 && (!aligned(a->x) || a->x_stride % 16 != 0 || (a->rows > 1 && a->x_stride < padded(a->K)))))
        return SD_ERR_INVALID_ARGUMENT;
    if (a->K > MAX_K || a->rows > 0x7fffff00LL || a->N > 0x7fffff00) return SD_ERR_UNSUPPORTED_SHAPE;   // rounded up to tiles, both stay in 32 bits
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    Int8Params p{};
    p.M = (int)a->rows; p.outs = a->swiglu ? a->N / 2 : a->N; p.K = a->K;
    p.x_scale = a->x_scale; p.w_scale = a->weight_scale;
    p.bias = a->bias; p.bias_f32 = a->bias_type == SD_F32;
    p.y = a->y; p.y_stride = a->y_stride; p.out_f32 = a->y_type == SD_F32;
    const bool token = token_takes(a);
    bool chained = a->chained != 0;
    Int8TokenParams t{};
    t.W = reinterpret_cast<const signed char*>(a->weight); t.w_stride = a->weight_stride;
    if (token_fuses(a)) {
        t.o = p; t.x = a->x; t.x_stride = a->x_stride;
        return token_rows<__nv_bfloat16>(t, a->swiglu != 0, chained, stream);
    }
    const void* q = a->x;
    long long q_stride = a->x_stride;
    const bool quantized = a->x_type == SD_I8;
    if (!quantized) {
        if (!a->scratch || !aligned(a->scratch) || a->scratch_bytes < sd_int8_linear_scratch_bytes(a)) return SD_ERR_BUFFER_TOO_SMALL;
        sd_quantize_rows_args r{};
        r.rows = a->rows; r.K = a->K; r.x_type = a->x_type; r.x = a->x; r.x_stride = a->x_stride;
        r.q = a->scratch; r.q_stride = padded(a->K);
        r.scale = reinterpret_cast<float*>(reinterpret_cast<char*>(a->scratch) + q_bytes(a));
        const int e = quantize(&r, chained, stream);
        if (e != SD_OK) return e;
        q = r.q; q_stride = r.q_stride; p.x_scale = r.scale;
        chained = true;
    }
    if (token) {
        t.o = p; t.x = q; t.x_stride = q_stride;
        return token_rows<signed char>(t, a->swiglu != 0, chained, stream);
    }
    return matmul(p, a, q, q_stride, chained, stream);
}

int sd_sample_tokens(const sd_sample_tokens_args* a, void* stream_) {
    if (!a || a->rows <= 0 || a->V <= 0 || !a->logits || !a->uniform || !a->tokens ||
        (a->logits_type != SD_BF16 && a->logits_type != SD_F32) || !aligned(a->logits, a->logits_type == SD_F32 ? 4 : 2))
        return SD_ERR_INVALID_ARGUMENT;
    if (a->V > SAMPLE_MAX_VOCAB || a->rows > (0x7fffffffLL >> 3)) return SD_ERR_UNSUPPORTED_SHAPE;
    SampleParams p{};
    p.V = a->V;
    p.logits = a->logits; p.stride = a->stride; p.uniform = a->uniform;
    p.temperature_row = a->temperature_row; p.top_k_row = a->top_k_row; p.top_p_row = a->top_p_row; p.min_p_row = a->min_p_row;
    // a number counts as its FP32 value, as in a tensor of settings: both give the same tokens
    p.temperature = (float)a->temperature; p.top_p = (float)a->top_p; p.min_p = (float)a->min_p; p.top_k = a->top_k;
    p.empty_token = a->empty_token;
    p.tokens = reinterpret_cast<long long*>(a->tokens);
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    return a->logits_type == SD_F32 ? sample<float>(p, a->rows, stream) : sample<__nv_bfloat16>(p, a->rows, stream);
}

}  // extern "C"
