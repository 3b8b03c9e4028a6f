// Operator-level entry points of matrices in 4 bits: b200_op_pack4, b200_op_unpack4, b200_op_dense4.
#include <algorithm>

#include "kernels_product4.cuh"
#include "op_product.h"
#include "with_type.h"

namespace {

using namespace b200;

int check_four(const char* who, int rows, int cols, int type, int by_column) {
    if (rows < 0 || cols < 1) return fail(B200_ERR_ARG, "%s: %d rows of %d", who, rows, cols);
    if (by_column != 0 && by_column != 1) return fail(B200_ERR_ARG, "%s: by_column is %d", who, by_column);
    if (!is_float(type)) return fail(B200_ERR_UNSUPPORTED, "%s: type %d", who, type);
    return 0;
}
// Rows of codes along `n`, and their scales.
int check_codes(const char* who, const char* what, const void* at, int64_t ld, int64_t rows, int64_t n, const void* scale) {
    if (!at || !scale) return fail(B200_ERR_ARG, "%s: %s or its scales are NULL", who, what);
    if ((uintptr_t)at % 16 || ld % 16 || (uintptr_t)scale % 16) return fail(B200_ERR_ARG, "%s: rows of %s, or its scales, do not start on 16 bytes", who, what);
    if (ld < (n + 31) / 32 * 16 || ld > INT64_MAX / 8 / (rows > 0 ? rows : 1))
        return fail(B200_ERR_ARG, "%s: ld of %s is %lld bytes, with rows of %lld codes", who, what, (long long)ld, (long long)n);
    return 0;
}
// How elements lie in rows (kFourEach).
int way_of(const void* at, int64_t ld, int cols, int type) {
    const uintptr_t places = (uintptr_t)at | (uintptr_t)(ld * type_bytes(type));
    return cols % 16 == 0 && places % 32 == 0 ? 2 : cols % 8 == 0 && places % 16 == 0 ? 1 : 0;
}
template <class F>
void with_way(int way, F f) {
    if (way == 2)
        f(std::integral_constant<int, 2>{});
    else if (way == 1)
        f(std::integral_constant<int, 1>{});
    else
        f(std::integral_constant<int, 0>{});
}
// CTAs for `places` of a thread each, kFourAhead at a time
unsigned ctas_for(int64_t places) {
    constexpr int64_t each = kFourThreads * kFourAhead;
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((places + each - 1) / each, kSms * 8));
}
dim3 column_grid(int64_t columns, int64_t groups) { return dim3((unsigned)((columns + 63) / 64), (unsigned)std::min<int64_t>((groups + 3) / 4, 65535)); }

// ---- products

// Which tile: by what each way costs in ns, from the launch to the first stage, a stage (256 of k), the rest of each tile after the first; rounds of tiles
// being whole.  Fitted to layers in bf16 without a residual.  With either tile, 16 to 131072 rows, 256 to 4096 inputs, 64 to 2048 outputs: of 225 such layers the choice is
// the quicker one, or within 2 %, in 223 (the worst, 16384 rows 256 -> 1024, 16.1 us for 15.0); with a residual in 216 (22.6 for 20.5 there), of 220 with results in fp32 in 215
// (19.7 for 17.0).  Us, 128 x 128 and 256 x 256 of a pair, in brackets with a residual: 300 rows 2048 -> 1024 8.1 and 10.1 (8.8 and 11.1), 5003 rows 10.8 and 11.2 of
// 1024 inputs (13.5 and 14.2), 14.7 and 14.1 of 2048 (15.6 and 15.9), 16384 rows 2048 -> 2048 47.4 and 35.2 (52.8 and 42.1), 131072 rows 1024 -> 64 19.5 and 20.0 (22.1 and
// 23.3), 2048 -> 1024 172 and 126 (202 and 159).
struct Way {
    int columns, rows, units, start, stage, tile;
};
constexpr Way kWays[] = {{256, 256, kSms / 2, 6600, 290, 1500}, {128, 128, kSms, 4500, 290, 850}};
int columns_of(int64_t m, int64_t n, int64_t blocks) {
    int best = 0;
    int64_t least = INT64_MAX;
    for (const Way& w : kWays) {
        const int64_t tiles = ((m + w.rows - 1) / w.rows) * ((n + w.columns - 1) / w.columns), rounds = (tiles + w.units - 1) / w.units;
        const int64_t cost = w.start + rounds * blocks * w.stage + (rounds - 1) * w.tile;
        if (cost < least) least = cost, best = w.columns;
    }
    return best;
}

int make_codes_map(CUtensorMap* map, const void* at, int64_t ld, int64_t rows, int64_t n, int box_rows) {
    const Encode encode = encoder();
    if (!encode) return fail(B200_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t bytes = (cuuint64_t)((n + 31) / 32 * 16), size[2] = {bytes, (cuuint64_t)rows}, stride[1] = {rows == 1 ? bytes : (cuuint64_t)ld};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, each[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(at), size, stride, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) on %lld rows of %lld codes, %lld bytes apart", (int)rc, (long long)rows, (long long)n, (long long)ld);
    return 0;
}
// Tiles of scales as a stack of matrices: 128 words a tile, in boxes of two side by side by `up`.
int make_scales_map(CUtensorMap* map, const void* at, int64_t rows, int64_t n, int up) {
    const Encode encode = encoder();
    if (!encode) return fail(B200_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t across = (cuuint64_t)((n + 127) / 128), size[3] = {128, across, (cuuint64_t)((rows + 127) / 128)}, stride[2] = {512, across * 512};
    const cuuint32_t box[3] = {128, 2, (cuuint32_t)up}, each[3] = {1, 1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(at), size, stride, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) on scales of %lld rows of %lld codes", (int)rc, (long long)rows, (long long)n);
    return 0;
}

template <int BN, bool PAIR, bool ADDS>
int launch_product(const b200_dense4_op* op, ProductArgs p, cudaStream_t stream) {
    using T = Tile4<BN, PAIR, ADDS>;
    p.tiles_m = (int)((p.m + T::kRows - 1) / T::kRows);
    p.tiles_n = (int)((p.n + BN - 1) / BN);
    if ((int64_t)p.tiles_m * p.tiles_n > INT32_MAX) return fail(B200_ERR_UNSUPPORTED, "op_dense4: %lld rows, %lld out are too many", (long long)p.m, (long long)p.n);
    CUtensorMap a, b, a_scale, b_scale, d{}, r{};
    if (int rc = make_codes_map(&a, op->x, op->ldx, p.m, p.k, 128)) return rc;
    if (int rc = make_codes_map(&b, op->w, op->ldw, p.n, p.k, T::kOwnColumns)) return rc;
    if (int rc = make_scales_map(&a_scale, op->x_scale, p.m, p.k, 1)) return rc;
    if (int rc = make_scales_map(&b_scale, op->w_scale, p.n, p.k, T::kScaleTiles)) return rc;
    if (p.boxes) {
        if (int rc = make_result_map(&d, p.d, p.d_type, p.ldd, p.m, p.n, 1, 64)) return rc;
        if (p.residual)
            if (int rc = make_result_map(&r, p.residual, p.d_type, p.ldr, p.m, p.n, 1, 64)) return rc;
    }
    auto kernel = product4_kernel<BN, PAIR, ADDS>;
    static std::atomic<uint64_t> allowed;  // a bit per device
    int device = 0;
    OP_CK(cudaGetDevice(&device));
    if (device >= 64 || !(allowed >> device & 1)) {
        OP_CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)T::kShared));
        if (device < 64) allowed |= (uint64_t)1 << device;
    }
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, units = PAIR ? kSms / 2 : kSms;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(std::min(tiles, units) * (PAIR ? 2 : 1)));
    config.blockDim = dim3(T::kThreads);
    config.dynamicSmemBytes = T::kShared;
    config.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {PAIR ? 2u : 1u, 1, 1};
    config.attrs = &attr;
    config.numAttrs = 1;
    OP_CK(cudaLaunchKernelEx(&config, kernel, a, b, a_scale, b_scale, d, r, p));
    return 0;
}

template <int R>
int launch_few(const b200_dense4_op* op, cudaStream_t stream) {
    const FourScales s{(op->in + 31ll) / 32};
    const int64_t shared = R * s.groups * 33;
    static std::atomic<uint64_t> allowed;
    int device = 0;
    OP_CK(cudaGetDevice(&device));
    if (device >= 64 || !(allowed >> device & 1)) {
        OP_CK(cudaFuncSetAttribute(dense4_few_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewFourBytes / 32 * 33));
        if (device < 64) allowed |= (uint64_t)1 << device;
    }
    dense4_few_kernel<R><<<(unsigned)std::min<int64_t>((op->out + 7ll) / 8, kSms * 4), 256, (size_t)shared, stream>>>(*op, s);
    OP_CK(cudaGetLastError());
    return 0;
}

}  // namespace

extern "C" {

int b200_op_pack4(int device, void* stream, const b200_pack4_op* op) {
    const char* who = "op_pack4";
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_four(who, op->rows, op->cols, op->x_type, op->by_column)) return rc;
    if (op->rows == 0) return 0;
    const int64_t rows = op->by_column ? op->cols : op->rows, n = op->by_column ? op->rows : op->cols;
    if (int rc = check_matrix(who, "x", op->x, op->ldx, op->rows, op->cols, op->x_type)) return rc;
    if (int rc = check_codes(who, "q", op->q, op->ldq, rows, n, op->scale)) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const FourScales scales{(n + 31) / 32};
    with_float(op->x_type, [&](auto x) {
        using T = decltype(x);
        if (op->by_column)
            pack4_columns_kernel<T><<<column_grid((rows + 127) / 128 * 128, scales.groups), kFourThreads, 0, s>>>(*op, scales);
        else
            with_way(way_of(op->x, op->ldx, op->cols, op->x_type), [&](auto w) {
                pack4_rows_kernel<T, w()><<<ctas_for((rows + 127) / 128 * 128 * scales.across() * 128 / kFourEach<w()>), kFourThreads, 0, s>>>(*op, scales);
            });
    });
    OP_CK(cudaGetLastError());
    return 0;
}

int b200_op_unpack4(int device, void* stream, const b200_unpack4_op* op) {
    const char* who = "op_unpack4";
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_four(who, op->rows, op->cols, op->y_type, op->by_column)) return rc;
    if (op->rows == 0) return 0;
    const int64_t rows = op->by_column ? op->cols : op->rows, n = op->by_column ? op->rows : op->cols;
    if (int rc = check_codes(who, "q", op->q, op->ldq, rows, n, op->scale)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->cols, op->y_type)) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const FourScales scales{(n + 31) / 32};
    with_float(op->y_type, [&](auto y) {
        using T = decltype(y);
        if (op->by_column)
            unpack4_columns_kernel<T><<<column_grid(rows, scales.groups), kFourThreads, 0, s>>>(*op, scales);
        else
            with_way(way_of(op->y, op->ldy, op->cols, op->y_type), [&](auto w) {
                unpack4_rows_kernel<T, w()><<<ctas_for(rows * ((op->cols + kFourEach<w()> - 1ll) / kFourEach<w()>)), kFourThreads, 0, s>>>(*op, scales);
            });
    });
    OP_CK(cudaGetLastError());
    return 0;
}

int b200_op_dense4(int device, void* stream, const b200_dense4_op* op) {
    const char* who = "op_dense4";
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->rows < 0 || op->in < 1 || op->out < 1) return fail(B200_ERR_ARG, "%s: %d rows, %d in, %d out", who, op->rows, op->in, op->out);
    if (!is_float(op->y_type)) return fail(B200_ERR_UNSUPPORTED, "%s: type %d", who, op->y_type);
    if (!is_act(op->act)) return fail(B200_ERR_ARG, "%s: %d names no activation", who, op->act);
    if (op->rows == 0) return 0;
    if (int rc = check_codes(who, "x", op->x, op->ldx, op->rows, op->in, op->x_scale)) return rc;
    if (int rc = check_codes(who, "w", op->w, op->ldw, op->out, op->in, op->w_scale)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->out, op->y_type)) return rc;
    if (op->residual)
        if (int rc = check_matrix(who, "residual", op->residual, op->ldr, op->rows, op->out, op->y_type)) return rc;
    if (op->bias)
        if (int rc = check_floats(who, "bias", op->bias)) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int* word = gave_up_word(device);
    if (int rc = check_gave_up(who, word)) return rc;
    const int64_t bytes = (op->in + 31ll) / 32 * 32;  // of a row of x
    if (op->rows == 1 && bytes <= kFewFourBytes) return launch_few<1>(op, s);
    if (op->rows == 2 && 2 * bytes <= kFewFourBytes) return launch_few<2>(op, s);
    if (op->rows <= 4 && 4 * bytes <= kFewFourBytes) return launch_few<4>(op, s);
    if (op->rows <= kFewFourRows && kFewFourRows * bytes <= kFewFourBytes) return launch_few<kFewFourRows>(op, s);
    ProductArgs p{};
    p.m = op->rows, p.n = op->out, p.k = op->in;
    p.k_blocks = (int)((p.k + 255) / 256);
    p.bias = op->bias, p.residual = op->residual, p.ldr = op->ldr;
    p.d = op->y, p.ldd = op->ldy, p.d_type = op->y_type, p.act = op->act;
    p.gave_up = word;
    const int size = type_bytes(p.d_type);
    auto starts = [&](const void* at, int64_t ld) { return (uintptr_t)at % 16 == 0 && (p.m == 1 || ld * size % 16 == 0); };
    // (rows end on 16 bytes as well: boxes that were cut off inside 16 bytes would write into what lies behind the row)
    p.boxes = p.n * size % 16 == 0 && starts(p.d, p.ldd) && (!p.residual || starts(p.residual, p.ldr));
    if (columns_of(p.m, p.n, p.k_blocks) == 256) return p.residual ? launch_product<256, true, true>(op, p, s) : launch_product<256, true, false>(op, p, s);
    return p.residual ? launch_product<128, false, true>(op, p, s) : launch_product<128, false, false>(op, p, s);
}

}  // extern "C"
