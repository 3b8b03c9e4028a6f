// Operator-level entry points of dense layers: b200_op_dense and its gradient.
#include <algorithm>
#include <atomic>

#include "gave_up.h"
#include "kernels_few.cuh"
#include "kernels_product.cuh"
#include "kernels_rows.cuh"
#include "op_call.h"

namespace {

using namespace b200;

// A wait of a kernel before that gave up (Waits) is reported by the next call on its device.
int check_gave_up(const char* who, int* word) {
    if (!take_gave_up(word)) return 0;
    return fail(B200_ERR_STATE, "%s: a kernel of a call before on this device waited too long for its own copies or products; that call's outputs are not valid", who);
}

// ---- products

struct Operand {  // rows of `cols` consecutive elements
    const void* at;
    int64_t ld, rows, cols;
    int type;
    int64_t bytes_of_row() const { return ld * type_bytes(type); }
    bool aligned() const { return (uintptr_t)at % 16 == 0 && bytes_of_row() % 16 == 0; }
    int64_t copy_ld() const { return (cols * type_bytes(type) + 15) / 16 * 16 / type_bytes(type); }
    int64_t copy_bytes() const { return aligned() ? 0 : (rows * copy_ld() * type_bytes(type) + 255) / 256 * 256; }
};
Operand operand(const void* at, int64_t ld, int64_t rows, int64_t cols, int type) {
    Operand o{at, ld, rows, cols, type};
    if (rows == 1) o.ld = o.copy_ld();  // (there is no second row)
    return o;
}

struct Call {
    Operand a, b;
    bool a_across, b_across, codes;  // codes: a is an 8-bit checkpoint with a scale per k
    bool follows;                    // a kernel of the same call stands before it on the stream
    ProductArgs p;
    bool bytes() const { return a.type == B200_TYPE_E4M3 && !codes; }
    int block() const { return bytes() ? 128 : 64; }  // of k in a stage
};

// How a product is cut: into tiles of which width, and k into how many parts.  By what each way costs in clocks: a stage (128 bytes of
// k) of a tile, an item besides, a join (launch, and its bytes per clock), rounds of items being whole.  Fitted to times on a B200: of 33
// products of 16 to 65536 rows, timed with every width and up to ten numbers of parts, this choice is within 10 % of the best on all
// but two (us, it and the best: 16 x 2048 -> 1024 10.8 and 8.7, gradient of 256 x 256 weights from 16384 rows 17.4 and 15.2).
struct Plan {
    int columns;  // of a tile; from 256 on a pair's
    int parts, blocks;  // pieces of k and the stages of each
    int chains() const { return (blocks + kChainMost - 1) / kChainMost; }
    bool joined() const { return parts > 1 || chains() > 1; }
};
constexpr int kSms = 148;  // that products are cut for
constexpr int kPartsMost = 32, kJoin = 4500, kJoinBytes = 2500;
struct TileCost {
    int columns, rows, units, stage, stage_codes, item;
};
constexpr TileCost kTiles[] = {{512, 256, kSms / 2, 1226, 1403, 5500}, {256, 256, kSms / 2, 687, 1222, 900}, {128, 128, kSms, 650, 1000, 900}, {64, 128, kSms, 600, 950, 900}};
Plan reckoned_plan(const Call& c) {
    const int64_t blocks = (c.p.k + c.block() - 1) / c.block();
    Plan best{};
    double least = 1e300;
    for (const TileCost& t : kTiles) {
        if (t.columns == 64 && c.bytes()) continue;  // (boxes across are 128 columns there)
        const int64_t tiles = ((c.p.m + t.rows - 1) / t.rows) * ((c.p.n + t.columns - 1) / t.columns);
        const double stage = c.codes ? t.stage_codes : t.stage;
        for (int64_t parts = 1; parts <= std::min<int64_t>(kPartsMost, blocks); parts++) {
            if (parts > 1 && tiles * (parts - 1) >= 2 * t.units) break;
            const int64_t each = (blocks + parts - 1) / parts, rounds = (tiles * parts + t.units - 1) / t.units;
            const int64_t chains = (each + kChainMost - 1) / kChainMost;
            double cost = (double)rounds * (each * stage + t.item * (t.columns == 512 ? chains : 1));
            if (parts > 1 || chains > 1) cost += kJoin + 8.0 * parts * c.p.m * c.p.n / kJoinBytes;
            if (cost < least) least = cost, best = {t.columns, (int)((blocks + each - 1) / each), (int)each};
        }
    }
    return best;
}
// The same, from the last ones that this thread asked for (2 us to reckon, and a gradient asks six times).
Plan plan_of(const Call& c) {
    struct Known {
        int64_t m, n, k;
        int kind;
        Plan plan;
    };
    thread_local Known known[16] = {};
    const int kind = 1 + c.bytes() + 2 * c.codes;  // (0: a place that holds none)
    Known& at = known[(c.p.m * 7 + c.p.n * 3 + c.p.k + kind) & 15];
    if (at.kind != kind || at.m != c.p.m || at.n != c.p.n || at.k != c.p.k) at = {c.p.m, c.p.n, c.p.k, kind, reckoned_plan(c)};
    return at.plan;
}
int64_t parts_bytes(const Call& c, const Plan& plan) { return plan.joined() ? (int64_t)plan.parts * c.p.m * ((c.p.n + 7) / 8 * 8) * 4 : 0; }
int64_t call_bytes(const Call& c) { return c.a.copy_bytes() + c.b.copy_bytes() + (parts_bytes(c, plan_of(c)) + 255) / 256 * 256; }

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                            CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder() {
    static std::atomic<void*> found;
    if (!found) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult how;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how) == cudaSuccess && how == cudaDriverEntryPointSuccess) found = fn;
    }
    return reinterpret_cast<Encode>(found.load());
}
int make_map(CUtensorMap* map, const Operand& o, int box_cols, int box_rows, bool swizzled) {
    const Encode encode = encoder();
    if (!encode) return fail(B200_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t size[2] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows}, stride[1] = {(cuuint64_t)o.bytes_of_row()};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, each[2] = {1, 1};
    const CUtensorMapDataType type = o.type == B200_TYPE_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : o.type == B200_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult rc = encode(map, type, 2, const_cast<void*>(o.at), size, stride, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS)
        return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) on %lld rows of %lld, %lld bytes apart", (int)rc, (long long)o.rows, (long long)o.cols, (long long)o.bytes_of_row());
    return 0;
}

// The result, or its parts, as a stack of matrices, in boxes of 32 rows of 128 bytes.
int make_result_map(CUtensorMap* map, const void* at, int type, int64_t ld, int64_t rows, int64_t cols, int64_t count) {
    const Encode encode = encoder();
    if (!encode) return fail(B200_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t row = (cuuint64_t)(rows == 1 ? (cols * type_bytes(type) + 15) / 16 * 16 : ld * type_bytes(type));
    const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)count}, stride[2] = {row, (cuuint64_t)rows * (cuuint64_t)(count > 1 ? ld * type_bytes(type) : row)};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / type_bytes(type)), 32, 1}, each[3] = {1, 1, 1};
    const CUtensorMapDataType kind = type == B200_TYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == B200_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult rc = encode(map, kind, 3, const_cast<void*>(at), size, stride, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) on %lld rows of %lld, %lld apart", (int)rc, (long long)rows, (long long)cols, (long long)ld);
    return 0;
}

template <int BN, bool BYTES, bool A_ACROSS, bool B_ACROSS, bool CODES>
int launch(const Call& c, cudaStream_t stream) {
    constexpr bool PAIR = BN >= 256;
    using T = Tile<BN, PAIR, BYTES, A_ACROSS, B_ACROSS, CODES>;
    CUtensorMap a, b, d{}, r{};
    if (int rc = CODES ? make_map(&a, c.a, 128, 64, false) : A_ACROSS ? make_map(&a, c.a, T::kBlock, T::kBlock, true) : make_map(&a, c.a, T::kBlock, 128, true)) return rc;
    if (int rc = B_ACROSS ? make_map(&b, c.b, T::kBlock, T::kBlock, true) : make_map(&b, c.b, T::kBlock, T::kOwnColumns, true)) return rc;
    if (c.p.parts) {
        if (int rc = make_result_map(&d, c.p.parts, B200_TYPE_F32, c.p.ldp, c.p.m, c.p.ldp, c.p.parts_n)) return rc;
    } else if (c.p.boxes) {
        if (int rc = make_result_map(&d, c.p.d, c.p.d_type, c.p.ldd, c.p.m, c.p.n, 1)) return rc;
        if (c.p.residual)
            if (int rc = make_result_map(&r, c.p.residual, c.p.d_type, c.p.ldr, c.p.m, c.p.n, 1)) return rc;
    }
    auto kernel = product_kernel<BN, PAIR, BYTES, A_ACROSS, B_ACROSS, CODES>;
    static std::atomic<uint64_t> allowed;  // a bit per device
    int device = 0;
    OP_CK(cudaGetDevice(&device));
    if (device >= 64 || !(allowed >> device & 1)) {
        OP_CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)T::kShared));
        if (device < 64) allowed |= (uint64_t)1 << device;
    }
    const int64_t items = (int64_t)c.p.tiles_m * c.p.tiles_n * c.p.parts_n, units = PAIR ? kSms / 2 : kSms;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(std::min(items, units) * (PAIR ? 2 : 1)));
    config.blockDim = dim3(T::kThreads);
    config.dynamicSmemBytes = T::kShared;
    config.stream = stream;
    cudaLaunchAttribute attrs[2] = {};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim = {PAIR ? 2u : 1u, 1, 1};
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = c.follows ? 2 : 1;
    OP_CK(cudaLaunchKernelEx(&config, kernel, a, b, d, r, c.p));
    return 0;
}
template <bool BYTES, bool A_ACROSS, bool B_ACROSS, bool CODES>
int launch_columns(const Call& c, int columns, cudaStream_t stream) {
    if (columns == 512) return launch<512, BYTES, A_ACROSS, B_ACROSS, CODES>(c, stream);
    if (columns == 256) return launch<256, BYTES, A_ACROSS, B_ACROSS, CODES>(c, stream);
    if constexpr (!BYTES)
        if (columns == 64) return launch<64, BYTES, A_ACROSS, B_ACROSS, CODES>(c, stream);
    return launch<128, BYTES, A_ACROSS, B_ACROSS, CODES>(c, stream);
}

// An operand whose rows do not start on 16 bytes is copied first: the copy moves less than the product does.
int align(Operand& o, char*& space, cudaStream_t stream) {
    if (o.aligned()) return 0;
    void* to = space;
    space += o.copy_bytes();
    const int64_t pieces = o.rows * (o.copy_ld() * type_bytes(o.type) / 16), grid = (pieces + 256 * kAlignPieces - 1) / (256 * kAlignPieces);
    if (grid > INT32_MAX) return fail(B200_ERR_UNSUPPORTED, "too many elements in rows that do not start on 16 bytes");
    align_rows_kernel<<<(unsigned)grid, 256, 0, stream>>>(static_cast<const uint8_t*>(o.at), o.bytes_of_row(), static_cast<uint4*>(to), o.rows, o.cols * type_bytes(o.type));
    OP_CK(cudaGetLastError());
    o.ld = o.copy_ld();
    o.at = to;
    return 0;
}

int run_product(Call c, char* space, cudaStream_t stream) {
    const Plan plan = plan_of(c);
    if (int rc = align(c.a, space, stream)) return rc;
    if (int rc = align(c.b, space, stream)) return rc;
    ProductArgs& p = c.p;
    const int rows = plan.columns >= 256 ? 256 : 128;
    p.tiles_m = (int)((p.m + rows - 1) / rows);
    p.tiles_n = (int)((p.n + plan.columns - 1) / plan.columns);
    p.k_blocks = (int)((p.k + c.block() - 1) / c.block());
    p.blocks_per_item = plan.blocks;
    p.parts_n = plan.parts;
    p.ldp = (p.n + 7) / 8 * 8;
    p.chain = (plan.blocks + plan.chains() - 1) / plan.chains();
    p.parts = plan.joined() ? reinterpret_cast<float*>(space) : nullptr;
    p.form_type = c.b.type == B200_TYPE_BF16;
    const int size = type_bytes(p.d_type);
    auto starts = [&](const void* at, int64_t ld) { return (uintptr_t)at % 16 == 0 && (p.m == 1 || ld * size % 16 == 0); };
    // (rows end on 16 bytes as well: boxes that were cut off inside 16 bytes wrote into what lies behind the row)
    p.boxes = p.parts || (p.n * size % 16 == 0 && starts(p.d, p.ldd) && (!p.residual || starts(p.residual, p.ldr)));
    const int rc = c.bytes()    ? launch_columns<true, false, true, false>(c, plan.columns, stream)
                   : c.codes    ? launch_columns<false, true, true, true>(c, plan.columns, stream)
                   : c.a_across ? launch_columns<false, true, true, false>(c, plan.columns, stream)
                   : c.b_across ? launch_columns<false, false, true, false>(c, plan.columns, stream)
                                : launch_columns<false, false, false, false>(c, plan.columns, stream);
    if (rc) return rc;
    if (p.parts) {
        OP_CK(launch_step(true, c.bytes() ? join_kernel<true> : join_kernel<false>, (unsigned)((p.m * (p.ldp / 4) + 255) / 256), 256, 0, stream, p));
    }
    return 0;
}

// ---- the operators

// How dense_dz_kernel deals a matrix out.
struct DzShape {
    bool vec;
    int across, pieces;
    dim3 grid;
};
DzShape dz_shape(const b200_dense_grad_op* op) {
    auto on = [](const void* at, int64_t ld, int bytes, int to) { return ((uintptr_t)at | (uintptr_t)(ld * bytes)) % to == 0; };
    DzShape s;
    s.vec = op->out % 8 == 0 && on(op->dy, op->lddy, 2, 16) &&
            (op->act == B200_ACT_NONE || (op->y_type == B200_TYPE_E4M3 ? on(op->y, op->ldy, 1, 8) : on(op->y, op->ldy, 2, 16)));
    const int vectors = s.vec ? op->out / 8 : op->out;
    s.across = 1;
    while (s.across < 256 && s.across < vectors) s.across *= 2;
    const int ctas = (vectors + s.across - 1) / s.across, at_once = 256 / s.across * 4;
    // Few rows: one piece, whose sums are the result, and no second launch.  Many: as many pieces as run at once, two to an SM (5003 x 1024
    // with dz, and the parts' sums: four to an SM 10.8 + 5.6 us, three 11.3 + 8, two 8.9 + 5; 16384 x 1024: 23.4, 26.3, 21.5 + 6.7).
    s.pieces = op->rows <= 4 * at_once ? 1 : std::max(1, std::min(op->rows / at_once, std::max(1, kSms * 2 / ctas)));
    s.grid = dim3(ctas, s.pieces);
    return s;
}

int check_dense(const b200_dense_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->rows < 0 || op->in < 1 || op->out < 1) return fail(B200_ERR_ARG, "%s: %d rows, %d in, %d out", who, op->rows, op->in, op->out);
    if (!(is_16_bits(op->x_type) || op->x_type == B200_TYPE_E4M3) || !is_float(op->y_type))
        return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->x_type, op->y_type);
    if (!is_act(op->act)) return fail(B200_ERR_ARG, "%s: %d names no activation", who, op->act);
    return 0;
}

int check_dense_grad(const b200_dense_grad_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->rows < 0 || op->in < 1 || op->out < 1) return fail(B200_ERR_ARG, "%s: %d rows, %d in, %d out", who, op->rows, op->in, op->out);
    auto checkpoint = [&](int type) { return type == op->dy_type || (type == B200_TYPE_E4M3 && op->dy_type == B200_TYPE_BF16); };
    if (!is_16_bits(op->dy_type) || !checkpoint(op->x_type) || !checkpoint(op->y_type) || !(op->dw_type == B200_TYPE_F32 || op->dw_type == op->dy_type))
        return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d, %d, %d", who, op->dy_type, op->x_type, op->y_type, op->dw_type);
    if (!is_act(op->act)) return fail(B200_ERR_ARG, "%s: %d names no activation", who, op->act);
    return 0;
}

Call forward_call(const b200_dense_op* op) {
    Call c{};
    c.a = operand(op->x, op->ldx, op->rows, op->in, op->x_type);
    c.b = operand(op->w, op->ldw, op->in, op->out, op->x_type);
    c.b_across = true;
    ProductArgs& p = c.p;
    p.m = op->rows, p.n = op->out, p.k = op->in;
    if (op->x_type == B200_TYPE_E4M3) p.a_scale = op->x_scale, p.b_scale = op->w_scale;
    p.bias = op->bias, p.residual = op->residual, p.ldr = op->ldr;
    p.d = op->y, p.ldd = op->ldy, p.d_type = op->y_type, p.act = op->act;
    return c;
}
// Few rows: dense_few_kernel.
bool few_rows(const b200_dense_op* op) { return op->rows <= kFewRowsMost; }
template <class T, bool VEC>
int launch_few_typed(const b200_dense_op* op, cudaStream_t stream) {
    const int groups = (op->out + kFewColumns - 1) / kFewColumns;
    int ctas = 1;  // of a cluster: while there are SMs for them and enough of k
    while (ctas < kFewClusterMost && groups * ctas * 2 <= 2 * kSms && op->in / (ctas * 2) >= 2 * kFewStep) ctas *= 2;
    FewArgs f{*op, (op->in + ctas - 1) / ctas};
    f.slice = (f.slice + kFewStep - 1) / kFewStep * kFewStep;
    auto go = [&](auto kernel) {
        cudaLaunchConfig_t config{};
        config.gridDim = dim3((unsigned)(groups * ctas));
        config.blockDim = dim3(256);
        config.stream = stream;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {(unsigned)ctas, 1, 1};
        config.attrs = &attr;
        config.numAttrs = 1;
        return cudaLaunchKernelEx(&config, kernel, f);
    };
    OP_CK(op->rows == 1   ? go(dense_few_kernel<T, 1, VEC>)
          : op->rows == 2 ? go(dense_few_kernel<T, 2, VEC>)
          : op->rows <= 4 ? go(dense_few_kernel<T, 4, VEC>)
                          : go(dense_few_kernel<T, 8, VEC>));
    return 0;
}
template <class T>
int launch_few(const b200_dense_op* op, cudaStream_t stream) {
    constexpr int kBytes = 8 * sizeof(T);
    const bool vec = op->out % 8 == 0 && (uintptr_t)op->w % kBytes == 0 && op->ldw * sizeof(T) % kBytes == 0;
    return vec ? launch_few_typed<T, true>(op, stream) : launch_few_typed<T, false>(op, stream);
}

int64_t dense_bytes(const b200_dense_op* op) {
    if (few_rows(op)) return 0;
    const int64_t bytes = op->rows ? call_bytes(forward_call(op)) : 0;
    return bytes ? bytes + 256 : 0;
}
// g: dz, or dy where that is dz
Call dx_call(const b200_dense_grad_op* op, const void* g, int64_t ldg) {
    Call c{};
    c.a = operand(g, ldg, op->rows, op->out, op->dy_type);
    c.b = operand(op->w, op->ldw, op->in, op->out, op->dy_type);
    ProductArgs& p = c.p;
    p.m = op->rows, p.n = op->in, p.k = op->out;
    p.residual = op->dskip, p.ldr = op->ldskip;
    p.d = op->dx, p.ldd = op->lddx, p.d_type = op->dy_type;
    return c;
}
Call dw_call(const b200_dense_grad_op* op, const void* g, int64_t ldg) {
    Call c{};
    c.a = operand(op->x, op->ldx, op->rows, op->in, op->x_type);
    c.b = operand(g, ldg, op->rows, op->out, op->dy_type);
    c.a_across = c.b_across = true;
    c.codes = op->x_type == B200_TYPE_E4M3;
    ProductArgs& p = c.p;
    p.m = op->in, p.n = op->out, p.k = op->rows;
    if (c.codes) p.a_scale = op->x_scale;
    p.d = op->dw, p.ldd = op->lddw, p.d_type = op->dw_type;
    return c;
}

// Where the parts of a gradient's workspace begin, in bytes, behind its first multiple of 256.
struct GradSpace {
    bool dz_made;
    int64_t ldz, dz, sums, products, all;
};
GradSpace grad_space(const b200_dense_grad_op* op) {
    GradSpace s{};
    if (op->rows == 0) return s;
    auto next = [&](int64_t bytes) {
        const int64_t at = s.all;
        s.all += (bytes + 255) / 256 * 256;
        return at;
    };
    s.ldz = (op->out + 7) / 8 * 8;
    // (dz is dy without an activation, but for two products of one that does not start on 16 bytes)
    s.dz_made = (op->dx || op->dw) && (op->act != B200_ACT_NONE || !operand(op->dy, op->lddy, op->rows, op->out, op->dy_type).aligned());
    s.dz = next(s.dz_made ? op->rows * s.ldz * 2 : 0);
    const int pieces = dz_shape(op).pieces;
    s.sums = next(op->dbias && pieces > 1 ? (int64_t)pieces * op->out * 4 : 0);
    const void* g = s.dz_made ? nullptr : op->dy;  // (dz is aligned, as NULL is)
    const int64_t ldg = s.dz_made ? s.ldz : op->lddy;
    s.products = next(std::max(op->dx ? call_bytes(dx_call(op, g, ldg)) : 0, op->dw ? call_bytes(dw_call(op, g, ldg)) : 0));
    if (s.all) s.all += 256;
    return s;
}
char* aligned_space(void* workspace) { return reinterpret_cast<char*>(((uintptr_t)workspace + 255) & ~(uintptr_t)255); }

}  // namespace

extern "C" {

int b200_op_dense_workspace(const b200_dense_op* op, int64_t* bytes) {
    if (int rc = check_dense(op, "op_dense")) return rc;
    if (!bytes) return fail(B200_ERR_ARG, "op_dense: null result");
    *bytes = dense_bytes(op);
    return 0;
}

int b200_op_dense(int device, void* stream, const b200_dense_op* op) {
    const char* who = "op_dense";
    if (int rc = check_dense(op, who)) return rc;
    if (op->rows == 0) return 0;
    const bool packed = op->x_type == B200_TYPE_E4M3;
    if (int rc = check_matrix(who, "x", op->x, op->ldx, op->rows, op->in, op->x_type)) return rc;
    if (int rc = check_matrix(who, "w", op->w, op->ldw, op->in, op->out, op->x_type)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->out, op->y_type)) return rc;
    if (op->residual)
        if (int rc = check_matrix(who, "residual", op->residual, op->ldr, op->rows, op->out, op->y_type)) return rc;
    if (op->bias)
        if (int rc = check_floats(who, "bias", op->bias)) return rc;
    if (packed) {
        if (int rc = check_floats(who, "x_scale", op->x_scale)) return rc;
        if (int rc = check_floats(who, "w_scale", op->w_scale)) return rc;
    }
    if (int rc = check_workspace(who, op->workspace, op->workspace_bytes, dense_bytes(op))) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int* word = gave_up_word(device);
    if (int rc = check_gave_up(who, word)) return rc;
    if (few_rows(op)) return packed ? launch_few<e4m3>(op, s) : op->x_type == B200_TYPE_BF16 ? launch_few<bf16>(op, s) : launch_few<f16>(op, s);
    Call c = forward_call(op);
    c.p.gave_up = word;
    return run_product(c, aligned_space(op->workspace), s);
}

int b200_op_dense_backward_workspace(const b200_dense_grad_op* op, int64_t* bytes) {
    if (int rc = check_dense_grad(op, "op_dense_backward")) return rc;
    if (!bytes) return fail(B200_ERR_ARG, "op_dense_backward: null result");
    *bytes = grad_space(op).all;
    return 0;
}

int b200_op_dense_backward(int device, void* stream, const b200_dense_grad_op* op) {
    const char* who = "op_dense_backward";
    if (int rc = check_dense_grad(op, who)) return rc;
    const bool acts = op->act != B200_ACT_NONE;
    if (op->dw)
        if (int rc = check_matrix(who, "dw", op->dw, op->lddw, op->in, op->out, op->dw_type)) return rc;
    if (op->dbias)
        if (int rc = check_floats(who, "dbias", op->dbias)) return rc;
    const GradSpace space = grad_space(op);
    if (op->rows) {
        if (int rc = check_matrix(who, "dy", op->dy, op->lddy, op->rows, op->out, op->dy_type)) return rc;
        if (acts) {
            if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->out, op->y_type)) return rc;
            if (op->y_type == B200_TYPE_E4M3)
                if (int rc = check_floats(who, "y_scale", op->y_scale)) return rc;
        }
        if (op->dw) {
            if (int rc = check_matrix(who, "x", op->x, op->ldx, op->rows, op->in, op->x_type)) return rc;
            if (op->x_type == B200_TYPE_E4M3)
                if (int rc = check_floats(who, "x_scale", op->x_scale)) return rc;
        }
        if (op->dx) {
            if (int rc = check_matrix(who, "dx", op->dx, op->lddx, op->rows, op->in, op->dy_type)) return rc;
            if (int rc = check_matrix(who, "w", op->w, op->ldw, op->in, op->out, op->dy_type)) return rc;
            if (op->dskip)
                if (int rc = check_matrix(who, "dskip", op->dskip, op->ldskip, op->rows, op->in, op->dy_type)) return rc;
        }
        if (int rc = check_workspace(who, op->workspace, op->workspace_bytes, space.all)) return rc;
    }
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (op->rows == 0) {
        if (op->dw) OP_CK(cudaMemset2DAsync(op->dw, op->lddw * type_bytes(op->dw_type), 0, (size_t)op->out * type_bytes(op->dw_type), op->in, s));
        if (op->dbias) OP_CK(cudaMemsetAsync(op->dbias, 0, (size_t)op->out * 4, s));
        return 0;
    }
    int* word = gave_up_word(device);
    if (int rc = check_gave_up(who, word)) return rc;
    char* base = aligned_space(op->workspace);
    void* dz = space.dz_made ? base + space.dz : nullptr;
    const DzShape g = dz_shape(op);
    float* sums = !op->dbias ? nullptr : g.pieces == 1 ? op->dbias : reinterpret_cast<float*>(base + space.sums);
    bool beside = false;  // the last kernel so far neither writes what the next product reads nor the other way round
    if (dz || sums) {
        auto go = [&](auto d, auto y) {
            using TD = decltype(d);
            using TY = decltype(y);
            if (g.vec)
                dense_dz_kernel<TD, TY, 8><<<g.grid, 256, 0, s>>>(*op, static_cast<TD*>(dz), space.ldz, sums, g.across);
            else
                dense_dz_kernel<TD, TY, 1><<<g.grid, 256, 0, s>>>(*op, static_cast<TD*>(dz), space.ldz, sums, g.across);
        };
        if (op->dy_type == B200_TYPE_F16)
            go(f16{}, f16{});
        else if (op->y_type == B200_TYPE_E4M3)
            go(bf16{}, e4m3{});
        else
            go(bf16{}, bf16{});
        OP_CK(cudaGetLastError());
        beside = sums && g.pieces > 1;
        if (beside) OP_CK(launch_step(true, add_parts_kernel, (op->out + 31) / 32, kAddThreads, 0, s, sums, g.pieces, op->out, op->dbias));
    }
    const void* gradient = dz ? dz : op->dy;
    const int64_t ld_gradient = dz ? space.ldz : op->lddy;
    if (op->dx) {
        Call c = dx_call(op, gradient, ld_gradient);
        c.follows = dz || sums;
        c.p.beside = beside && c.a.aligned() && c.b.aligned();
        c.p.gave_up = word;
        beside = call_bytes(c) == 0;
        if (int rc = run_product(c, base + space.products, s)) return rc;
    }
    if (op->dw) {
        Call c = dw_call(op, gradient, ld_gradient);
        c.follows = dz || sums || op->dx;
        c.p.beside = beside && c.a.aligned() && c.b.aligned();
        c.p.gave_up = word;
        if (int rc = run_product(c, base + space.products, s)) return rc;
    }
    return 0;
}

}  // extern "C"
