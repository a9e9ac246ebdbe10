// C ABI of the dense operators (declared in include/alpha_dense.h): argument checks, the layout of the caller's workspace
// and the sequence of kernels. Everything is enqueued on streams[0]; nothing is allocated, freed or synchronised here.
#include "dense_common.hpp"

#include <cmath>
#include <cstdarg>
#include <cstdio>

using namespace alpha;

namespace {

thread_local char g_err[256] = "";

int fail(const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return ALPHA_DENSE_EINVAL;
}

int hip_status(hipError_t e, const char *what)
{
    if (e == hipSuccess) return 0;
    snprintf(g_err, sizeof(g_err), "%s: %s", what, hipGetErrorString(e));
    return (int)e;
}

inline long round8(long n) { return (n + 7) & ~7l; }
inline size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
inline size_t size_of(int type) { return type == ALPHA_DENSE_F32 ? 4 : 2; }

// Takes blocks of the caller's workspace one after another; with no workspace it only counts.
struct Scratch {
    char *base;
    size_t at;
    explicit Scratch(void *p) : base(static_cast<char *>(p)), at(0) {}
    template <typename T> T *take(size_t bytes)
    {
        T *p = base && bytes ? reinterpret_cast<T *>(base + at) : nullptr;
        at += round256(bytes);
        return p;
    }
};

bool sizes_served(int type, int64_t N, int64_t IC, int64_t OC, int pair = 1)
{
    if (type != ALPHA_DENSE_F32 && type != ALPHA_DENSE_BF16) return false;
    if (N < 0 || N >= (1 << 30) || IC < 0 || OC < 0 || IC > (1 << 22) || pair * OC > (1 << 22)) return false;   // (a pair's deltaZ lie side by side)
    // packed tensors of at most 2^34 elements: their 16-byte chunks are counted in 31 bits
    return N * round8(IC) < (1l << 34) && 2 * N * round8(OC) < (1l << 34) && OC * round8(IC) < (1l << 34);
}

int check_call(const char *fn, const int64_t *streams, int length, int type, int N, int IC, int OC, int act, float k, const void *workspace,
               int64_t bytes, int64_t need)   // need < 0: sizes not served
{
    if (streams == nullptr || length < 1) return fail("%s: empty stream array", fn);
    if (type != ALPHA_DENSE_F32 && type != ALPHA_DENSE_BF16) return fail("%s: unknown element type %d", fn, type);
    if (act < ALPHA_DENSE_ACT_NONE || act > ALPHA_DENSE_ACT_SIGMOID) return fail("%s: unknown activation %d", fn, act);
    if (act == ALPHA_DENSE_ACT_LEAKY_RELU && !std::isfinite(k)) return fail("%s: slope k is not finite", fn);
    if (need < 0) return fail("%s: size out of range (N %d, IC %d, OC %d)", fn, N, IC, OC);
    if (need > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) || bytes < need))
        return fail("%s: workspace is null, not 256-byte aligned or too small (%lld of %lld bytes)", fn, (long long)bytes, (long long)need);
    return 0;
}

// A stream of another device than the current one would launch kernels there on memory of here.
int check_device(const char *fn, hipStream_t s)
{
    if (s == nullptr) return 0;
    hipDevice_t of = 0;
    int current = 0;
    hipError_t e = hipStreamGetDevice(s, &of);
    if (e == hipSuccess) e = hipGetDevice(&current);
    if (e != hipSuccess) return hip_status(e, fn);
    if ((int)of != current) return fail("%s: the stream belongs to device %d, the current device is %d", fn, (int)of, current);
    return 0;
}

// a matrix argument: NULL (where allowed) or aligned to its element, with a row stride the kernels can take
int check_matrix(const char *fn, const char *name, const void *p, int64_t stride, int rows, int cols, int type, bool needed)
{
    if (p == nullptr) return needed && rows > 0 && cols > 0 ? fail("%s: %s is null", fn, name) : 0;
    if (reinterpret_cast<uintptr_t>(p) & (size_of(type) - 1)) return fail("%s: %s is not aligned to its element", fn, name);
    if (stride < cols || stride > (1 << 22)) return fail("%s: %s_stride %lld is out of range (row length %d)", fn, name, (long long)stride, cols);
    return 0;
}

int check_vector(const char *fn, const char *name, const void *p, int type)
{
    if (reinterpret_cast<uintptr_t>(p) & (size_of(type) - 1)) return fail("%s: %s is not aligned to its element", fn, name);
    return 0;
}

// Two outputs, or an output and an input, of one address. (Interleaved column ranges of one buffer are legal, so ranges are not compared.)
int check_distinct(const char *fn, const void *const *outputs, int n_out, const void *const *inputs, int n_in)
{
    for (int i = 0; i < n_out; i++) {
        if (outputs[i] == nullptr) continue;
        for (int j = i + 1; j < n_out; j++)
            if (outputs[i] == outputs[j]) return fail("%s: two outputs share an address", fn);
        for (int j = 0; j < n_in; j++)
            if (outputs[i] == inputs[j]) return fail("%s: an output shares its address with an input", fn);
    }
    return 0;
}

// Clipping: a tensor written twice would be scaled twice, or by two workgroups at a time; one that is another's source, before or
// after it is read. A filter of 2^17 bits (16 KB on the stack) leaves few addresses to look for one by one.
int check_clip_lists(const char *fn, int count, const int64_t *lengths, const void *const *src, void *const *dst)
{
    uint64_t seen[2048] = {};
    auto place = [](const void *p) { return (unsigned)((reinterpret_cast<uintptr_t>(p) * 0x9e3779b97f4a7c15ull) >> 47); };
    auto look = [&](const void *p, int end, int except) {
        if ((seen[place(p) >> 6] >> (place(p) & 63) & 1) == 0) return -1;
        for (int j = 0; j < end; j++)
            if (j != except && lengths[j] > 0 && dst[j] == p) return j;
        return -1;
    };
    for (int i = 0; i < count; i++) {
        if (lengths[i] == 0) continue;
        const int j = look(dst[i], i, i);
        if (j >= 0) return fail("%s: dst[%d] and dst[%d] share an address", fn, j, i);
        seen[place(dst[i]) >> 6] |= 1ull << (place(dst[i]) & 63);
    }
    for (int i = 0; i < count; i++) {
        if (lengths[i] == 0 || src[i] == dst[i]) continue;
        const int j = look(src[i], count, i);
        if (j >= 0) return fail("%s: dst[%d] shares its address with src[%d]", fn, j, i);
    }
    return 0;
}

#define TRY(call)             \
    do {                      \
        if (int rc_ = (call)) \
            return rc_;       \
    } while (0)

// May the tile kernel read the tensor in place? fp32 always; bf16, whose 128-bit loads go straight to LDS, rows of whole 16-byte
// chunks.
bool in_place(int type, const void *p, int64_t stride, int cols)
{
    return type == ALPHA_DENSE_F32 || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride & 7) == 0 && (cols & 7) == 0);
}

// Room for a packed [rows, cols] tensor, whether the call will need it or not: the workspace does not depend on addresses. fp32
// needs it only for a pair of filters, whose row strides have to be one.
size_t packed_bytes(int type, long rows, long cols, int pair = 0)
{
    return type == ALPHA_DENSE_F32 && !pair ? 0 : (size_t)rows * round8(cols) * size_of(type);
}

// One source of an operand of the tile kernel, packed if it has to be.
int operand(const char *fn, hipStream_t s, int type, const void *p, int64_t stride, long rows, int cols, void *room, bool pack, DenseOperand &o, int which)
{
    o.p[which] = pack ? room : p;
    o.ld = pack ? round8(cols) : stride;
    if (!pack) return 0;
    return hip_status(launch_dense_pack(s, type == ALPHA_DENSE_F32, p, stride, rows, cols, room, o.ld), fn);
}

int quads_aligned(int type, std::initializer_list<const void *> p, std::initializer_list<int64_t> strides)
{
    const uintptr_t mask = type == ALPHA_DENSE_F32 ? 15 : 7;
    for (const void *q : p)
        if (reinterpret_cast<uintptr_t>(q) & mask) return 0;
    for (int64_t x : strides)
        if (x & 3) return 0;
    return 1;
}


// ---- workspaces: the same sequence of blocks for the query (base NULL) and the call --------------------------------
struct ForwardRoom {
    DenseForm form;
    void *X, *W[2];
    float *pieces;
    size_t piece_bytes, total;
};
ForwardRoom forward_room(int type, int N, int IC, int OC, int gated, void *base)
{
    Scratch ws(base);
    ForwardRoom r{};
    r.form = dense_forward_form(type == ALPHA_DENSE_F32, gated, N, OC, IC);
    if (r.form != DENSE_TILES_FORM) {   // operands as they are
        if (r.form == DENSE_FEW_ROWS) r.piece_bytes = dense_few_rows_piece_bytes(type == ALPHA_DENSE_F32, gated, N, OC, IC);
        r.pieces = ws.take<float>(r.piece_bytes);
        r.total = ws.at;
        return r;
    }
    r.X = ws.take<void>(packed_bytes(type, N, IC));
    for (int i = 0; i < (gated ? 2 : 1); i++) r.W[i] = ws.take<void>(packed_bytes(type, OC, IC, gated));
    r.piece_bytes = dense_product_piece_bytes(N, OC, IC, type == ALPHA_DENSE_F32, 1, gated);
    r.pieces = ws.take<float>(r.piece_bytes);
    r.total = ws.at;
    return r;
}

struct BackwardRoom {
    char *delta;
    void *X, *W[2];
    float *sums, *pieces;
    size_t piece_bytes, total;
};
BackwardRoom backward_room(int type, int N, int IC, int OC, int gated, void *base)
{
    Scratch ws(base);
    BackwardRoom r{};
    const int pair = gated ? 2 : 1;
    r.delta = ws.take<char>((size_t)N * pair * round8(OC) * size_of(type));
    r.X = ws.take<void>(packed_bytes(type, N, IC));
    for (int i = 0; i < pair; i++) r.W[i] = ws.take<void>(packed_bytes(type, OC, IC, gated));
    r.sums = ws.take<float>(dense_delta_sum_bytes(N, OC, gated));
    // two small products are one launch, so their pieces are there at a time
    struct Pieces {
        size_t small, tiles;
    };
    auto pieces = [&](int a_t, int M, int N, int K, int sources) {
        const int f32 = type == ALPHA_DENSE_F32;
        if (dense_small_preferred(f32, a_t, M, N, K, sources)) return Pieces{dense_small_piece_bytes(f32, M, N, K, sources), 0};
        return Pieces{0, dense_product_piece_bytes(M, N, K, f32, sources, 0)};
    };
    // a gated pair's filter gradients are one stacked product, or one of them alone
    const Pieces x = pieces(0, N, IC, OC, pair), w = pieces(1, OC, IC, N, 1), both = gated ? pieces(1, (int)round8(OC) + OC, IC, N, 1) : Pieces{0, 0};
    r.piece_bytes = std::max({x.small + std::max(w.small, both.small), x.tiles, w.tiles, both.tiles});
    r.pieces = ws.take<float>(r.piece_bytes);
    r.total = ws.at;
    return r;
}

// Forward, plain and gated.
int forward(const char *fn, hipStream_t s, int type, int gated, const void *X, int64_t ldX, const void *W, int64_t ldW, const void *W2, int64_t ldW2,
            const DenseEpilogue &ep, int N, int IC, int OC, const ForwardRoom &room)
{
    if (room.form != DENSE_TILES_FORM) {
        DenseFewRows a{};
        a.X = X;
        a.ldX = ldX;
        a.W = W;
        a.ldW = ldW;
        a.W2 = W2;
        a.ldW2 = ldW2;
        a.f32 = type == ALPHA_DENSE_F32;
        a.gated = gated;
        a.M = N;
        a.N = OC;
        a.K = IC;
        a.ep = ep;
        a.pieces = room.pieces;
        a.piece_bytes = room.piece_bytes;
        return hip_status(room.form == DENSE_FEW_ROWS ? launch_dense_few_rows(s, a) : launch_dense_short(s, a), fn);
    }
    DenseProduct p{};
    p.sources = 1;
    p.gated = gated;
    p.M = N;
    p.N = OC;
    p.K = IC;
    p.f32 = type == ALPHA_DENSE_F32;
    p.ep = ep;
    p.pieces = room.pieces;
    p.piece_bytes = room.piece_bytes;
    if (IC > 0) {
        TRY(operand(fn, s, type, X, ldX, N, IC, room.X, !in_place(type, X, ldX, IC), p.A, 0));
        const bool pack = !in_place(type, W, ldW, IC) || (gated && (!in_place(type, W2, ldW2, IC) || ldW != ldW2));
        TRY(operand(fn, s, type, W, ldW, OC, IC, room.W[0], pack, p.B, 0));
        if (gated) TRY(operand(fn, s, type, W2, ldW2, OC, IC, room.W[1], pack, p.B, 1));
    }
    return hip_status(launch_dense_product(s, p), fn);
}

struct BackwardCall {
    const void *dY, *Z, *U, *X, *W[2];
    int64_t ld_dY, ldZ, ldU, ldX, ldW[2];
    void *dX, *dW[2], *dB[2];
    int64_t ld_dX, ld_dW[2];
};

int backward(const char *fn, hipStream_t s, int type, int gated, const BackwardCall &c, int act, float k, int N, int IC, int OC, const BackwardRoom &room)
{
    const bool want_x = c.dX != nullptr && N > 0 && IC > 0, want_w = (c.dW[0] || c.dW[1]) && OC > 0 && IC > 0;
    const bool products = want_x || want_w;
    const int pair = gated ? 2 : 1;

    // deltaZ and its sums
    DenseDelta d{};
    d.dY = c.dY;
    d.Z = c.Z;
    d.U = c.U;
    d.ldY = c.ld_dY;
    d.ldZ = c.ldZ;
    d.ldU = c.ldU;
    d.f32 = type == ALPHA_DENSE_F32;
    d.act = act;
    d.gated = gated;
    d.slope = k;
    d.rows = N;
    d.cols = OC;
    d.ld = round8(OC);
    d.ld2 = pair * d.ld;
    d.dB = c.dB[0];
    d.dB2 = c.dB[1];
    d.sums = room.sums;
    DenseOperand delta{};
    if (!gated && act == ALPHA_DENSE_ACT_NONE && in_place(type, c.dY, c.ld_dY, OC)) {   // deltaZ is deltaY
        delta.p[0] = c.dY;
        delta.ld = c.ld_dY;
    } else {
        if (products) d.dst = room.delta;
        if (products && gated) d.dst2 = room.delta ? room.delta + d.ld * size_of(type) : nullptr;
        delta.p[0] = room.delta;
        delta.p[1] = gated && room.delta ? room.delta + d.ld * size_of(type) : nullptr;
        delta.ld = d.ld2;
    }
    if (d.dst || d.dB || d.dB2) TRY(hip_status(launch_dense_delta(s, d), fn));

    DenseProduct p{};
    p.f32 = d.f32;
    p.pieces = room.pieces;
    p.piece_bytes = room.piece_bytes;
    DenseProduct small_x{};      // waits for deltaW
    if (want_x) {   // deltaX[n, ic] = sum over oc (and over both filters)
        p.A = delta;
        p.sources = pair;
        p.b_t = 1;
        p.M = N;
        p.N = IC;
        p.K = OC;
        p.ep = DenseEpilogue{};
        p.ep.Y = c.dX;
        p.ep.ldY = c.ld_dX;
        p.ep.vec = quads_aligned(type, {c.dX}, {c.ld_dX});
        const bool small = dense_small_preferred(p.f32, 0, p.M, p.N, p.K, p.sources);
        if (OC > 0) {
            const bool strides = gated && c.ldW[0] != c.ldW[1];
            const bool pack = strides || (!small && (!in_place(type, c.W[0], c.ldW[0], IC) || (gated && !in_place(type, c.W[1], c.ldW[1], IC))));
            for (int i = 0; i < pair; i++) TRY(operand(fn, s, type, c.W[i], c.ldW[i], OC, IC, room.W[i], pack, p.B, i));
        }
        if (!small) TRY(hip_status(launch_dense_product(s, p), fn));
        else if (want_w) small_x = p;
        else TRY(hip_status(launch_dense_small(s, &p, nullptr), fn));
    }
    const DenseProduct *waiting = small_x.M > 0 ? &small_x : nullptr;
    if (want_w) {   // deltaW[oc, ic] = sum over n; both filters' as one product over the pair's columns
        p.A = delta;
        p.B = DenseOperand{};
        p.sources = 1;
        p.a_t = p.b_t = 1;
        p.N = IC;
        p.K = N;
        p.ep = DenseEpilogue{};
        const int first = c.dW[0] ? 0 : 1;
        p.A.p[0] = delta.p[first];
        p.ep.Y = c.dW[first];
        p.ep.ldY = c.ld_dW[first];
        p.M = OC;
        p.ep.vec = quads_aligned(type, {c.dW[first]}, {c.ld_dW[first]});
        if (c.dW[0] && c.dW[1]) {
            p.M = (int)round8(OC) + OC;
            p.ep.rows1 = OC;
            p.ep.row2 = (int)round8(OC);
            p.ep.Y2 = c.dW[1];
            p.ep.ldY2 = c.ld_dW[1];
            p.ep.vec = p.ep.vec && quads_aligned(type, {c.dW[1]}, {c.ld_dW[1]});
        }
        const bool small = dense_small_preferred(p.f32, 1, p.M, p.N, p.K, 1);
        if (N > 0) TRY(operand(fn, s, type, c.X, c.ldX, N, IC, room.X, !small && !in_place(type, c.X, c.ldX, IC), p.B, 0));
        if (small) {
            TRY(hip_status(launch_dense_small(s, waiting, &p), fn));
        } else {
            if (waiting) TRY(hip_status(launch_dense_small(s, waiting, nullptr), fn));
            TRY(hip_status(launch_dense_product(s, p), fn));
        }
    }
    return 0;
}

}  // namespace

extern "C" {

#define ALPHA_EXPORT __attribute__((visibility("default")))

ALPHA_EXPORT const char *alpha_dense_last_error(void) { return g_err; }

ALPHA_EXPORT int64_t alpha_matMul_fused_workspace(int type, int N, int IC, int OC)
{
    return sizes_served(type, N, IC, OC) ? (int64_t)forward_room(type, N, IC, OC, 0, nullptr).total : -1;
}

ALPHA_EXPORT int alpha_matMul_fused(const int64_t *streams, int length, int type, const void *X, int64_t X_stride, const void *W, int64_t W_stride,
                                    const void *Bias, int act, float k, const void *R, int64_t R_stride, void *Z, int64_t Z_stride, void *Y,
                                    int64_t Y_stride, int N, int IC, int OC, void *workspace, int64_t workspace_bytes)
{
    const char *fn = __func__;
    const bool served = sizes_served(type, N, IC, OC);
    const ForwardRoom room = served ? forward_room(type, N, IC, OC, 0, workspace) : ForwardRoom{};
    TRY(check_call(fn, streams, length, type, N, IC, OC, act, k, workspace, workspace_bytes, served ? (int64_t)room.total : -1));
    TRY(check_matrix(fn, "X", X, X_stride, N, IC, type, true));
    TRY(check_matrix(fn, "W", W, W_stride, OC, IC, type, true));
    TRY(check_vector(fn, "Bias", Bias, type));
    TRY(check_matrix(fn, "R", R, R_stride, N, OC, type, false));
    TRY(check_matrix(fn, "Z", Z, Z_stride, N, OC, type, false));
    TRY(check_matrix(fn, "Y", Y, Y_stride, N, OC, type, true));
    const void *out[] = {Y, Z}, *in[] = {X, W, Bias, workspace}, *z[] = {Z}, *r[] = {R};
    TRY(check_distinct(fn, out, 2, in, 4));
    TRY(check_distinct(fn, z, 1, r, 1));
    if (R != nullptr && R == Y && R_stride != Y_stride) return fail("%s: Y is R with another stride", fn);
    if (N == 0 || OC == 0) return 0;
    hipStream_t s = reinterpret_cast<hipStream_t>((intptr_t)streams[0]);
    TRY(check_device(fn, s));
    DenseEpilogue ep{};
    ep.bias = Bias;
    ep.R = R;
    ep.ldR = R_stride;
    ep.Z = Z;
    ep.ldZ = Z_stride;
    ep.Y = Y;
    ep.ldY = Y_stride;
    ep.act = act;
    ep.slope = k;
    ep.vec = quads_aligned(type, {Bias, R, Z, Y}, {R ? R_stride : 0, Z ? Z_stride : 0, Y_stride});
    return forward(fn, s, type, 0, X, X_stride, W, W_stride, nullptr, 0, ep, N, IC, OC, room);
}

ALPHA_EXPORT int64_t alpha_dmatMul_fused_workspace(int type, int N, int IC, int OC)
{
    return sizes_served(type, N, IC, OC) ? (int64_t)backward_room(type, N, IC, OC, 0, nullptr).total : -1;
}

ALPHA_EXPORT int alpha_dmatMul_fused(const int64_t *streams, int length, int type, const void *deltaY, int64_t deltaY_stride, const void *Z,
                                     int64_t Z_stride, int act, float k, const void *X, int64_t X_stride, const void *W, int64_t W_stride,
                                     void *deltaX, int64_t deltaX_stride, void *deltaW, int64_t deltaW_stride, void *deltaB, int N, int IC, int OC,
                                     void *workspace, int64_t workspace_bytes)
{
    const char *fn = __func__;
    const bool served = sizes_served(type, N, IC, OC);
    const BackwardRoom room = served ? backward_room(type, N, IC, OC, 0, workspace) : BackwardRoom{};
    TRY(check_call(fn, streams, length, type, N, IC, OC, act, k, workspace, workspace_bytes, served ? (int64_t)room.total : -1));
    TRY(check_matrix(fn, "deltaY", deltaY, deltaY_stride, N, OC, type, true));
    if (act != ALPHA_DENSE_ACT_NONE) TRY(check_matrix(fn, "Z", Z, Z_stride, N, OC, type, true));
    TRY(check_matrix(fn, "X", X, X_stride, N, IC, type, deltaW != nullptr));
    TRY(check_matrix(fn, "W", W, W_stride, OC, IC, type, deltaX != nullptr));
    TRY(check_matrix(fn, "deltaX", deltaX, deltaX_stride, N, IC, type, false));
    TRY(check_matrix(fn, "deltaW", deltaW, deltaW_stride, OC, IC, type, false));
    TRY(check_vector(fn, "deltaB", deltaB, type));
    const void *out[] = {deltaX, deltaW, deltaB}, *in[] = {deltaY, act != ALPHA_DENSE_ACT_NONE ? Z : nullptr, X, W, workspace};
    TRY(check_distinct(fn, out, 3, in, 5));
    hipStream_t s = reinterpret_cast<hipStream_t>((intptr_t)streams[0]);
    TRY(check_device(fn, s));
    BackwardCall c{};
    c.dY = deltaY;
    c.ld_dY = deltaY_stride;
    if (act != ALPHA_DENSE_ACT_NONE) {
        c.Z = Z;
        c.ldZ = Z_stride;
    }
    c.X = X;
    c.ldX = X_stride;
    c.W[0] = W;
    c.ldW[0] = W_stride;
    c.dX = deltaX;
    c.ld_dX = deltaX_stride;
    c.dW[0] = deltaW;
    c.ld_dW[0] = deltaW_stride;
    c.dB[0] = deltaB;
    return backward(fn, s, type, 0, c, act, k, N, IC, OC, room);
}

ALPHA_EXPORT int64_t alpha_gatedMatMul_workspace(int type, int N, int IC, int OC)
{
    return sizes_served(type, N, IC, OC, 2) ? (int64_t)forward_room(type, N, IC, OC, 1, nullptr).total : -1;
}

ALPHA_EXPORT int alpha_gatedMatMul(const int64_t *streams, int length, int type, const void *X, int64_t X_stride, const void *Wg, int64_t Wg_stride,
                                   const void *Bg, const void *Wu, int64_t Wu_stride, const void *Bu, int act, float k, void *G, int64_t G_stride,
                                   void *U, int64_t U_stride, void *H, int64_t H_stride, int N, int IC, int OC, void *workspace,
                                   int64_t workspace_bytes)
{
    const char *fn = __func__;
    const bool served = sizes_served(type, N, IC, OC, 2);
    const ForwardRoom room = served ? forward_room(type, N, IC, OC, 1, workspace) : ForwardRoom{};
    TRY(check_call(fn, streams, length, type, N, IC, OC, act, k, workspace, workspace_bytes, served ? (int64_t)room.total : -1));
    TRY(check_matrix(fn, "X", X, X_stride, N, IC, type, true));
    TRY(check_matrix(fn, "Wg", Wg, Wg_stride, OC, IC, type, true));
    TRY(check_matrix(fn, "Wu", Wu, Wu_stride, OC, IC, type, true));
    TRY(check_vector(fn, "Bg", Bg, type));
    TRY(check_vector(fn, "Bu", Bu, type));
    TRY(check_matrix(fn, "G", G, G_stride, N, OC, type, false));
    TRY(check_matrix(fn, "U", U, U_stride, N, OC, type, false));
    TRY(check_matrix(fn, "H", H, H_stride, N, OC, type, true));
    const void *out[] = {H, G, U}, *in[] = {X, Wg, Wu, Bg, Bu, workspace};
    TRY(check_distinct(fn, out, 3, in, 6));
    if (N == 0 || OC == 0) return 0;
    hipStream_t s = reinterpret_cast<hipStream_t>((intptr_t)streams[0]);
    TRY(check_device(fn, s));
    DenseEpilogue ep{};
    ep.bias = Bg;
    ep.bias2 = Bu;
    ep.Z = G;
    ep.ldZ = G_stride;
    ep.Z2 = U;
    ep.ldZ2 = U_stride;
    ep.Y = H;
    ep.ldY = H_stride;
    ep.act = act;
    ep.slope = k;
    ep.vec = quads_aligned(type, {Bg, Bu, G, U, H}, {G ? G_stride : 0, U ? U_stride : 0, H_stride});
    return forward(fn, s, type, 1, X, X_stride, Wg, Wg_stride, Wu, Wu_stride, ep, N, IC, OC, room);
}

ALPHA_EXPORT int64_t alpha_dgatedMatMul_workspace(int type, int N, int IC, int OC)
{
    return sizes_served(type, N, IC, OC, 2) ? (int64_t)backward_room(type, N, IC, OC, 1, nullptr).total : -1;
}

ALPHA_EXPORT int alpha_dgatedMatMul(const int64_t *streams, int length, int type, const void *deltaH, int64_t deltaH_stride, const void *G,
                                    int64_t G_stride, const void *U, int64_t U_stride, int act, float k, const void *X, int64_t X_stride,
                                    const void *Wg, int64_t Wg_stride, const void *Wu, int64_t Wu_stride, void *deltaX, int64_t deltaX_stride,
                                    void *deltaWg, int64_t deltaWg_stride, void *deltaWu, int64_t deltaWu_stride, void *deltaBg, void *deltaBu,
                                    int N, int IC, int OC, void *workspace, int64_t workspace_bytes)
{
    const char *fn = __func__;
    const bool served = sizes_served(type, N, IC, OC, 2);
    const BackwardRoom room = served ? backward_room(type, N, IC, OC, 1, workspace) : BackwardRoom{};
    TRY(check_call(fn, streams, length, type, N, IC, OC, act, k, workspace, workspace_bytes, served ? (int64_t)room.total : -1));
    TRY(check_matrix(fn, "deltaH", deltaH, deltaH_stride, N, OC, type, true));
    TRY(check_matrix(fn, "G", G, G_stride, N, OC, type, true));
    TRY(check_matrix(fn, "U", U, U_stride, N, OC, type, true));
    TRY(check_matrix(fn, "X", X, X_stride, N, IC, type, deltaWg != nullptr || deltaWu != nullptr));
    TRY(check_matrix(fn, "Wg", Wg, Wg_stride, OC, IC, type, deltaX != nullptr));
    TRY(check_matrix(fn, "Wu", Wu, Wu_stride, OC, IC, type, deltaX != nullptr));
    TRY(check_matrix(fn, "deltaX", deltaX, deltaX_stride, N, IC, type, false));
    TRY(check_matrix(fn, "deltaWg", deltaWg, deltaWg_stride, OC, IC, type, false));
    TRY(check_matrix(fn, "deltaWu", deltaWu, deltaWu_stride, OC, IC, type, false));
    TRY(check_vector(fn, "deltaBg", deltaBg, type));
    TRY(check_vector(fn, "deltaBu", deltaBu, type));
    const void *out[] = {deltaX, deltaWg, deltaWu, deltaBg, deltaBu}, *in[] = {deltaH, G, U, X, Wg, Wu, workspace};
    TRY(check_distinct(fn, out, 5, in, 7));
    hipStream_t s = reinterpret_cast<hipStream_t>((intptr_t)streams[0]);
    TRY(check_device(fn, s));
    BackwardCall c{};
    c.dY = deltaH;
    c.ld_dY = deltaH_stride;
    c.Z = G;
    c.ldZ = G_stride;
    c.U = U;
    c.ldU = U_stride;
    c.X = X;
    c.ldX = X_stride;
    c.W[0] = Wg;
    c.ldW[0] = Wg_stride;
    c.W[1] = Wu;
    c.ldW[1] = Wu_stride;
    c.dX = deltaX;
    c.ld_dX = deltaX_stride;
    c.dW[0] = deltaWg;
    c.ld_dW[0] = deltaWg_stride;
    c.dW[1] = deltaWu;
    c.ld_dW[1] = deltaWu_stride;
    c.dB[0] = deltaBg;
    c.dB[1] = deltaBu;
    return backward(fn, s, type, 1, c, act, k, N, IC, OC, room);
}

ALPHA_EXPORT int64_t alpha_gradClip_workspace(int count, const int64_t *lengths)
{
    if (count < 0 || (count > 0 && lengths == nullptr)) return -1;
    int64_t pieces = 0;
    for (int i = 0; i < count; i++) {
        if (lengths[i] < 0 || lengths[i] > (1l << 40)) return -1;
        pieces += grad_pieces(lengths[i]);
    }
    return (int64_t)round256((size_t)pieces * sizeof(double));
}

ALPHA_EXPORT int alpha_gradClip(const int64_t *streams, int length, int count, const int *types, const int64_t *lengths, const void *const *src,
                                void *const *dst, float max_norm, float eps, float *norm_c, void *workspace, int64_t workspace_bytes)
{
    const char *fn = __func__;
    if (streams == nullptr || length < 1) return fail("%s: empty stream array", fn);
    if (count < 0 || (count > 0 && (types == nullptr || lengths == nullptr || src == nullptr))) return fail("%s: null tensor list", fn);
    if (!std::isfinite(max_norm) || !std::isfinite(eps) || max_norm < 0.f || eps < 0.f || !(max_norm + eps > 0.f))
        return fail("%s: max_norm %g and eps %g must be finite, not negative and not both zero", fn, (double)max_norm, (double)eps);
    if (norm_c == nullptr || (reinterpret_cast<uintptr_t>(norm_c) & 3)) return fail("%s: norm_c is null or not aligned", fn);
    const int64_t need = alpha_gradClip_workspace(count, lengths);
    if (need < 0) return fail("%s: a tensor's length is out of range", fn);
    if (need > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < need))
        return fail("%s: workspace is null, not 256-byte aligned or too small (%lld of %lld bytes)", fn, (long long)workspace_bytes, (long long)need);
    for (int i = 0; i < count; i++) {
        if (types[i] != ALPHA_DENSE_F32 && types[i] != ALPHA_DENSE_BF16) return fail("%s: unknown element type %d of tensor %d", fn, types[i], i);
        if (lengths[i] == 0) continue;
        if (src[i] == nullptr || (reinterpret_cast<uintptr_t>(src[i]) & (size_of(types[i]) - 1))) return fail("%s: src[%d] is null or not aligned to its element", fn, i);
        if (dst != nullptr && (dst[i] == nullptr || (reinterpret_cast<uintptr_t>(dst[i]) & (size_of(types[i]) - 1))))
            return fail("%s: dst[%d] is null or not aligned to its element", fn, i);
    }
    if (dst != nullptr) TRY(check_clip_lists(fn, count, lengths, src, dst));
    hipStream_t s = reinterpret_cast<hipStream_t>((intptr_t)streams[0]);
    TRY(check_device(fn, s));
    return hip_status(launch_grad_clip(s, count, types, lengths, src, dst, max_norm, eps, norm_c, static_cast<double *>(workspace)), fn);
}

}  // extern "C"
