// Host side of the embedding operators declared in include/browservec_hip.h:
// handles, argument checks, launches (bv_linear.hip, bv_linear_q8.hip,
// bv_attention.hip, bv_attention_local.hip, bv_rows.hip, bv_add_norm.hip).
#include "bv_embed.h"
#include "bv_host.h"

#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <vector>

using namespace bvk;

struct bv_embed {
    std::mutex mu;
    bv_device *dev = nullptr;
    hipStream_t own = nullptr, stream = nullptr;
    void *zeros = nullptr;  // 256 bytes of zeros
    // Workspaces of each stream that needed one, the last of a stream's in
    // use; a capture has its own, since its graph may run beside the stream's
    // other work and other graphs.  All stay until the handle goes: kernels that
    // still run, and graphs, hold their addresses.  Each is at least one and a
    // half times the one before.
    struct Workspace {
        hipStream_t stream;
        unsigned long long capture;  // 0: none
        void *p;
        size_t cap;
    };
    std::vector<Workspace> ws;
};

namespace {

int embed_live(bv_embed *e) {
    if (e->dev->lost) return fail(BV_E_DEVICE_LOST, "GPU device lost; re-create the store");
    HIPX(e->dev, hipSetDevice(e->dev->ordinal), "hipSetDevice");
    return BV_OK;
}

int embed_workspace(bv_embed *e, size_t bytes, void **out) {
    if (!bytes) return BV_OK;
    unsigned long long capture = 0;
    if (e->stream) {  // the null stream cannot be captured
        hipStreamCaptureStatus status;
        unsigned long long id = 0;
        HIPX(e->dev, hipStreamGetCaptureInfo(e->stream, &status, &id), "workspace");
        if (status == hipStreamCaptureStatusActive) capture = id + 1;
    }
    size_t had = 0;
    for (size_t i = e->ws.size(); i-- && !had;)
        if (e->ws[i].stream == e->stream && e->ws[i].capture == capture) {
            had = e->ws[i].cap;
            *out = e->ws[i].p;
        }
    if (bytes <= had) return BV_OK;
    bv_embed::Workspace w{e->stream, capture, nullptr, (std::max(bytes, had + had / 2) + 4095) & ~size_t(4095)};
    try {
        e->ws.reserve(e->ws.size() + 1);
    } catch (const std::bad_alloc &) {
        return fail(BV_E_OOM, "out of host memory");
    }
    // an allocation is no part of a capture: only the relaxed mode lets it pass
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    if (capture) HIPX(e->dev, hipThreadExchangeStreamCaptureMode(&mode), "workspace");
    const hipError_t err = hipMalloc(&w.p, w.cap);
    if (capture) (void)hipThreadExchangeStreamCaptureMode(&mode);
    HIPX(e->dev, err, "workspace");
    e->ws.push_back(w);
    *out = w.p;
    return BV_OK;
}

// Products of sizes and strides that fit 63 bits, so that no offset wraps.
bool fits(std::initializer_list<std::pair<uint64_t, uint64_t>> dims, uint64_t elem, uint64_t *bytes) {
    unsigned __int128 last = 0;
    for (const auto &d : dims) {
        if (d.first == 0) {
            *bytes = 0;
            return true;
        }
        last += (unsigned __int128)(d.first - 1) * d.second;
    }
    last = (last + 1) * elem;
    *bytes = (uint64_t)last;
    return last < ((unsigned __int128)1 << 62);
}

// The bytes an argument covers: `bytes` from p on, of them `width` at every
// `pitch`.  Heads have a second, finer pattern where tokens and heads lie at
// multiples of the smaller stride.
struct Span {
    const char *name;
    const void *p;
    uint64_t bytes;
    struct {
        uint64_t pitch, width;
    } at[2];
};
// Whether two arguments share memory.  Views of one buffer whose rows, or heads,
// lie side by side at the same pitch do not.
bool overlap(const Span &a, const Span &b) {
    const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    if (!a.bytes || !b.bytes || pa >= pb + b.bytes || pb >= pa + a.bytes) return false;
    for (const auto &x : a.at)
        for (const auto &y : b.at) {
            // one piece fits any pitch
            const uint64_t pitch = x.width == a.bytes ? y.pitch : y.width == b.bytes || x.pitch == y.pitch ? x.pitch : 0;
            if (!pitch) continue;
            const uint64_t d = pb >= pa ? (pb - pa) % pitch : (pitch - (pa - pb) % pitch) % pitch;
            if (d >= x.width && d + y.width <= pitch) return false;
        }
    return true;
}

uint64_t size_of(uint32_t dtype) { return dtype == BV_F32 ? 4 : dtype == BV_I8 ? 1 : 2; }

// before: the size that an earlier, shorter form of the struct has; what it lacks
// is 0.
template <class A>
int check_args(bv_embed *e, const A *given, A &a, const char *what, size_t before = sizeof(A)) {
    if (!e || !given) return fail(BV_E_INVALID, "%s: null argument", what);
    if (given->size != sizeof(A) && given->size != before)
        return fail(BV_E_INVALID, "%s: args.size is %u, not %zu", what, given->size, sizeof(A));
    memset(&a, 0, sizeof(A));
    memcpy(&a, given, given->size);
    return BV_OK;
}

// A matrix [rows][cols], its row stride filled in.
int check_matrix(const char *what, Span &s, const void *p, uint64_t rows, uint64_t cols, uint64_t &stride, uint64_t elem) {
    s.p = p;
    if (stride == 0) stride = cols;
    if (stride < cols)
        return fail(BV_E_INVALID, "%s: stride %llu of %s is shorter than its rows (%llu)", what, (unsigned long long)stride,
                    s.name, (unsigned long long)cols);
    if (!fits({{rows, stride}, {cols, 1}}, elem, &s.bytes)) return fail(BV_E_INVALID, "%s: %s is too large", what, s.name);
    if (s.bytes && !p) return fail(BV_E_INVALID, "%s: %s is null", what, s.name);
    if ((uintptr_t)p % elem) return fail(BV_E_INVALID, "%s: %s is not aligned to its type", what, s.name);
    s.at[0] = {stride * elem, cols * elem};
    return BV_OK;
}

// Heads [tokens][heads][d], both strides filled in, also those that a single
// token or head leaves without a meaning; of tokens and heads either may be the
// outer one.
int check_heads(const char *what, Span &s, const void *p, uint64_t tokens, uint64_t heads, uint64_t d, uint64_t &stride,
                uint64_t &head_stride, uint64_t elem) {
    s.p = p;
    if (tokens == 0 || heads == 0) return BV_OK;
    if (head_stride == 0 || heads == 1) head_stride = d;
    if (stride == 0 || tokens == 1) stride = heads * head_stride;
    const bool tokens_outer = head_stride >= d && (tokens <= 1 || stride >= (heads - 1) * head_stride + d);
    const bool heads_outer = stride >= d && (heads <= 1 || (unsigned __int128)head_stride >=
                                             (unsigned __int128)(tokens - 1) * stride + d);
    if (!tokens_outer && !heads_outer)
        return fail(BV_E_INVALID, "%s: %s: strides %llu and %llu make heads overlap", what, s.name,
                    (unsigned long long)stride, (unsigned long long)head_stride);
    if (!fits({{tokens, stride}, {heads, head_stride}, {d, 1}}, elem, &s.bytes))
        return fail(BV_E_INVALID, "%s: %s is too large", what, s.name);
    if (s.bytes && !p) return fail(BV_E_INVALID, "%s: %s is null", what, s.name);
    if ((uintptr_t)p % elem) return fail(BV_E_INVALID, "%s: %s is not aligned to its type", what, s.name);
    if (tokens == 1 || heads == 1) {  // the other's stride alone
        s.at[0] = {(heads == 1 ? stride : head_stride) * elem, d * elem};
        return BV_OK;
    }
    const uint64_t outer = tokens_outer ? stride : head_stride, inner = tokens_outer ? head_stride : stride;
    s.at[0] = {outer * elem, (((tokens_outer ? heads : tokens) - 1) * inner + d) * elem};
    if (outer % inner == 0) s.at[1] = {inner * elem, d * elem};
    return BV_OK;
}

int check_apart(const char *what, const Span &out, std::initializer_list<Span> ins) {
    for (const Span &in : ins)
        if (overlap(out, in)) return fail(BV_E_INVALID, "%s: %s overlaps %s", what, out.name, in.name);
    return BV_OK;
}

constexpr uint64_t TOKENS_MOST = 0x7fffffffull;  // int32 offsets

#define OK_OR_RETURN(expr)       \
    do {                         \
        const int _rc = (expr);  \
        if (_rc) return _rc;     \
    } while (0)

}  // namespace

// ---------------------------------------------------------------- handles --
extern "C" int bv_embed_create(bv_device *dev, bv_embed **out) {
    if (!dev || !out) return fail(BV_E_INVALID, "null argument");
    if (dev->lost) return fail(BV_E_DEVICE_LOST, "GPU device lost; re-create the store");
    HIPX(dev, hipSetDevice(dev->ordinal), "hipSetDevice");
    bv_embed *e = new (std::nothrow) bv_embed();
    if (!e) return fail(BV_E_OOM, "out of host memory");
    e->dev = dev;
    hipError_t err = hipStreamCreateWithFlags(&e->own, hipStreamNonBlocking);
    if (err == hipSuccess) err = hipMalloc(&e->zeros, 256);
    if (err == hipSuccess) err = hipMemset(e->zeros, 0, 256);
    if (err == hipSuccess) err = hipStreamSynchronize(nullptr);  // before any stream's first call
    if (err != hipSuccess) {
        if (e->zeros) (void)hipFree(e->zeros);
        if (e->own) (void)hipStreamDestroy(e->own);
        delete e;
        return hip_fail(dev, err, "bv_embed_create");
    }
    e->stream = e->own;
    *out = e;
    return BV_OK;
}

extern "C" int bv_embed_destroy(bv_embed *e) {
    if (!e) return BV_OK;
    (void)hipSetDevice(e->dev->ordinal);
    (void)hipDeviceSynchronize();
    for (const auto &w : e->ws) (void)hipFree(w.p);
    (void)hipFree(e->zeros);
    (void)hipStreamDestroy(e->own);
    delete e;
    return BV_OK;
}

extern "C" int bv_embed_set_stream(bv_embed *e, void *stream) {
    if (!e) return fail(BV_E_INVALID, "null handle");
    std::lock_guard<std::mutex> lock(e->mu);
    e->stream = (hipStream_t)stream;
    return BV_OK;
}

extern "C" int bv_embed_stream(bv_embed *e, void **stream) {
    if (!e || !stream) return fail(BV_E_INVALID, "null argument");
    *stream = e->stream;
    return BV_OK;
}

extern "C" int bv_embed_sync(bv_embed *e) {
    if (!e) return fail(BV_E_INVALID, "null handle");
    std::lock_guard<std::mutex> lock(e->mu);
    OK_OR_RETURN(embed_live(e));
    HIPX(e->dev, hipStreamSynchronize(e->stream), "sync");
    return BV_OK;
}

// ----------------------------------------------------------------- linear --
extern "C" int bv_embed_linear(bv_embed *e, const bv_embed_linear_args *args) {
    bv_embed_linear_args a;
    OK_OR_RETURN(check_args(e, args, a, "linear"));
    if (a.dtype != BV_F16 && a.dtype != BV_BF16)
        return fail(BV_E_UNSUPPORTED, "linear: dtype %u is not BV_F16 or BV_BF16", a.dtype);
    if (a.out_dtype != a.dtype && a.out_dtype != BV_F32)
        return fail(BV_E_UNSUPPORTED, "linear: out_dtype %u is neither dtype nor BV_F32", a.out_dtype);
    if (a.activation > BV_ACT_SILU) return fail(BV_E_INVALID, "linear: unknown activation %u", a.activation);
    const uint64_t in = 2, out = size_of(a.out_dtype);
    Span x{"x"}, w{"w"}, b{"bias"}, r{"residual"}, y{"y"};
    OK_OR_RETURN(check_matrix("linear", x, a.x, a.m, a.k, a.x_stride, in));
    OK_OR_RETURN(check_matrix("linear", w, a.w, a.n, a.k, a.w_stride, in));
    OK_OR_RETURN(check_matrix("linear", y, a.y, a.m, a.n, a.y_stride, out));
    if (a.bias) {
        uint64_t one = 0;
        OK_OR_RETURN(check_matrix("linear", b, a.bias, 1, a.n, one, in));
    }
    if (a.residual) {
        OK_OR_RETURN(check_matrix("linear", r, a.residual, a.m, a.n, a.residual_stride, out));
        const bool same = a.residual == a.y && a.residual_stride == a.y_stride;
        if (!same) OK_OR_RETURN(check_apart("linear", y, {r}));
    }
    OK_OR_RETURN(check_apart("linear", y, {x, w, b}));
    std::lock_guard<std::mutex> lock(e->mu);
    OK_OR_RETURN(embed_live(e));
    if (a.m == 0 || a.n == 0) return BV_OK;
    LinearArgs l{};
    l.dtype = (int)a.dtype;
    l.out_dtype = (int)a.out_dtype;
    l.act = (int)a.activation;
    l.m = a.m;
    l.n = a.n;
    l.k = a.k;
    l.x = a.x;
    l.w = a.w;
    l.bias = a.bias;
    l.residual = a.residual;
    l.y = a.y;
    l.ldx = a.x_stride;
    l.ldw = a.w_stride;
    l.ldr = a.residual_stride;
    l.ldy = a.y_stride;
    void *ws = nullptr;
    OK_OR_RETURN(embed_workspace(e, linear_workspace(l), &ws));
    HIPX(e->dev, launch_linear(l, ws, e->stream), "linear kernel");
    return BV_OK;
}

extern "C" int bv_embed_linear_q8(bv_embed *e, const bv_embed_linear_q8_args *args) {
    bv_embed_linear_q8_args a;
    OK_OR_RETURN(check_args(e, args, a, "linear_q8"));
    if (a.out_dtype > BV_BF16 || (a.bias && a.bias_dtype > BV_BF16)) return fail(BV_E_UNSUPPORTED, "linear_q8: unknown dtype");
    if (a.activation > BV_ACT_SILU) return fail(BV_E_INVALID, "linear_q8: unknown activation %u", a.activation);
    if (a.k > LINEAR_Q8_MAX_K)
        return fail(BV_E_UNSUPPORTED, "linear_q8: k %u exceeds %u, up to which sums of 32 bits are exact", a.k, LINEAR_Q8_MAX_K);
    const uint64_t out = size_of(a.out_dtype);
    Span x{"x"}, w{"w"}, sx{"x_scales"}, sw{"w_scales"}, b{"bias"}, r{"residual"}, y{"y"};
    OK_OR_RETURN(check_matrix("linear_q8", x, a.x, a.m, a.k, a.x_stride, 1));
    OK_OR_RETURN(check_matrix("linear_q8", w, a.w, a.n, a.k, a.w_stride, 1));
    OK_OR_RETURN(check_matrix("linear_q8", y, a.y, a.m, a.n, a.y_stride, out));
    uint64_t one = 0;
    OK_OR_RETURN(check_matrix("linear_q8", sx, a.x_scales, 1, a.m, one, 4));
    one = 0;
    OK_OR_RETURN(check_matrix("linear_q8", sw, a.w_scales, 1, a.n, one, 4));
    one = 0;
    if (a.bias) OK_OR_RETURN(check_matrix("linear_q8", b, a.bias, 1, a.n, one, size_of(a.bias_dtype)));
    if (a.residual) {
        OK_OR_RETURN(check_matrix("linear_q8", r, a.residual, a.m, a.n, a.residual_stride, out));
        const bool same = a.residual == a.y && a.residual_stride == a.y_stride;
        if (!same) OK_OR_RETURN(check_apart("linear_q8", y, {r}));
    }
    OK_OR_RETURN(check_apart("linear_q8", y, {x, w, sx, sw, b}));
    std::lock_guard<std::mutex> lock(e->mu);
    OK_OR_RETURN(embed_live(e));
    if (a.m == 0 || a.n == 0) return BV_OK;
    LinearQ8Args l{};
    l.out_dtype = (int)a.out_dtype;
    l.act = (int)a.activation;
    l.bias_dtype = (int)a.bias_dtype;
    l.m = a.m;
    l.n = a.n;
    l.k = a.k;
    l.x = (const int8_t *)a.x;
    l.w = (const int8_t *)a.w;
    l.x_scales = (const float *)a.x_scales;
    l.w_scales = (const float *)a.w_scales;
    l.bias = a.bias;
    l.residual = a.residual;
    l.y = a.y;
    l.ldx = a.x_stride;
    l.ldw = a.w_stride;
    l.ldr = a.residual_stride;
    l.ldy = a.y_stride;
    void *ws = nullptr;
    OK_OR_RETURN(embed_workspace(e, linear_q8_workspace(l), &ws));
    HIPX(e->dev, launch_linear_q8(l, ws, e->stream), "linear_q8 kernel");
    return BV_OK;
}

// ----------------------------------------------------------------- rotary --
extern "C" int bv_embed_rotary(bv_embed *e, const bv_embed_rotary_args *args) {
    bv_embed_rotary_args a;
    OK_OR_RETURN(check_args(e, args, a, "rotary"));
    if (a.dtype > BV_BF16) return fail(BV_E_UNSUPPORTED, "rotary: unknown dtype %u", a.dtype);
    if (a.rot_dim % 2 || a.rot_dim > a.head_dim)
        return fail(BV_E_INVALID, "rotary: rot_dim %u is not even or exceeds head_dim %u", a.rot_dim, a.head_dim);
    if (a.head_dim == 0 || a.heads_q == 0) return fail(BV_E_INVALID, "rotary: no heads");
    if ((uint64_t)a.head_dim > 65536 || (uint64_t)a.heads_q + a.heads_k > 65536)
        return fail(BV_E_UNSUPPORTED, "rotary: head_dim and heads are at most 65536");
    const uint64_t el = size_of(a.dtype);
    Span q{"q"}, k{"k"}, qo{"q_out"}, ko{"k_out"}, table{"table"}, pos{"positions"};
    OK_OR_RETURN(check_heads("rotary", q, a.q, a.tokens, a.heads_q, a.head_dim, a.q_stride, a.q_head_stride, el));
    OK_OR_RETURN(check_heads("rotary", qo, a.q_out, a.tokens, a.heads_q, a.head_dim, a.q_out_stride, a.q_out_head_stride, el));
    OK_OR_RETURN(check_heads("rotary", k, a.k, a.tokens, a.heads_k, a.head_dim, a.k_stride, a.k_head_stride, el));
    OK_OR_RETURN(check_heads("rotary", ko, a.k_out, a.tokens, a.heads_k, a.head_dim, a.k_out_stride, a.k_out_head_stride, el));
    uint64_t one = 0;
    OK_OR_RETURN(check_matrix("rotary", table, a.table, a.table_rows, a.rot_dim, one, 4));
    if (a.positions) {
        one = 0;
        OK_OR_RETURN(check_matrix("rotary", pos, a.positions, a.tokens, 1, one, 4));
    }
    const bool q_in = a.q == a.q_out && a.q_stride == a.q_out_stride && a.q_head_stride == a.q_out_head_stride;
    const bool k_in = a.k == a.k_out && a.k_stride == a.k_out_stride && a.k_head_stride == a.k_out_head_stride;
    if (!q_in) OK_OR_RETURN(check_apart("rotary", qo, {q}));
    if (!k_in) OK_OR_RETURN(check_apart("rotary", ko, {k}));
    OK_OR_RETURN(check_apart("rotary", qo, {k, ko, table, pos}));
    OK_OR_RETURN(check_apart("rotary", ko, {q, table, pos}));
    std::lock_guard<std::mutex> lock(e->mu);
    OK_OR_RETURN(embed_live(e));
    if (a.tokens == 0) return BV_OK;
    RotaryArgs r{};
    r.dtype = (int)a.dtype;
    r.interleaved = a.interleaved != 0;
    r.hq = a.heads_q;
    r.hk = a.heads_k;
    r.d = a.head_dim;
    r.rot = a.rot_dim;
    r.rows = a.table_rows;
    r.tokens = a.tokens;
    r.table = a.table;
    r.pos = a.positions;
    r.q = a.q;
    r.k = a.k;
    r.qo = a.q_out;
    r.ko = a.k_out;
    r.sq = a.q_stride;
    r.sqh = a.q_head_stride;
    r.sk = a.k_stride;
    r.skh = a.k_head_stride;
    r.sqo = a.q_out_stride;
    r.sqoh = a.q_out_head_stride;
    r.sko = a.k_out_stride;
    r.skoh = a.k_out_head_stride;
    HIPX(e->dev, launch_rotary(r, e->stream), "rotary kernel");
    return BV_OK;
}

extern "C" int bv_embed_rotary_table(const bv_embed_rotary_scaling *scaling, uint32_t table_rows, uint32_t rot_dim,
                                     float *table, uint64_t n_floats) {
    if (!scaling) return fail(BV_E_INVALID, "rotary table: null argument");
    if (scaling->size != sizeof(*scaling))
        return fail(BV_E_INVALID, "rotary table: scaling.size is %u, not %zu", scaling->size, sizeof(*scaling));
    const bv_embed_rotary_scaling s = *scaling;
    if (rot_dim % 2) return fail(BV_E_INVALID, "rotary table: rot_dim %u is not even", rot_dim);
    if (n_floats != (uint64_t)table_rows * rot_dim)
        return fail(BV_E_INVALID, "expected %llu floats, got %llu", (unsigned long long)((uint64_t)table_rows * rot_dim),
                    (unsigned long long)n_floats);
    if (n_floats == 0) return BV_OK;
    if (!table) return fail(BV_E_INVALID, "rotary table: table is null");
    if (s.kind > BV_ROTARY_PARTS) return fail(BV_E_INVALID, "rotary table: unknown scaling %u", s.kind);
    if (!(s.base > 0) || !std::isfinite(s.base)) return fail(BV_E_INVALID, "rotary table: base must be positive");
    if (s.kind != BV_ROTARY_NONE && (!(s.factor > 0) || !std::isfinite(s.factor)))
        return fail(BV_E_INVALID, "rotary table: factor must be positive");
    if (s.kind == BV_ROTARY_BASE && rot_dim <= 2)
        return fail(BV_E_INVALID, "rotary table: scaling the base needs a rot_dim above 2");
    if (s.kind == BV_ROTARY_PARTS &&
        (!(s.original_rows > 0) || !(s.high_turns > s.low_turns) || !std::isfinite(s.original_rows) ||
         !std::isfinite(s.high_turns) || !std::isfinite(s.low_turns)))
        return fail(BV_E_INVALID, "rotary table: parts need original_rows above 0 and high_turns above low_turns");
    if (!std::isfinite(s.magnitude)) return fail(BV_E_INVALID, "rotary table: magnitude is not finite");
    const double mag = s.magnitude == 0 ? 1.0 : s.magnitude;
    const double base = s.kind == BV_ROTARY_BASE ? s.base * std::pow(s.factor, rot_dim / (rot_dim - 2.0)) : s.base;
    for (uint32_t i = 0; i < rot_dim / 2; i++) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (s.kind == BV_ROTARY_LINEAR) f /= s.factor;
        if (s.kind == BV_ROTARY_PARTS) {
            const double turns = s.original_rows * f / (2 * M_PI);
            const double g = std::min(1.0, std::max(0.0, (turns - s.low_turns) / (s.high_turns - s.low_turns)));
            f *= g + (1 - g) / s.factor;
        }
        for (uint32_t p = 0; p < table_rows; p++) {
            float *at = table + (uint64_t)p * rot_dim + 2 * i;
            at[0] = (float)(mag * std::cos(p * f));
            at[1] = (float)(mag * std::sin(p * f));
        }
    }
    return BV_OK;
}

// -------------------------------------------------------------- attention --
extern "C" int bv_embed_attention(bv_embed *e, const bv_embed_attention_args *args) {
    bv_embed_attention_args a;
    static_assert(offsetof(bv_embed_attention_args, window) == BV_EMBED_ATTENTION_ARGS_V1, "the struct's first form");
    OK_OR_RETURN(check_args(e, args, a, "attention", BV_EMBED_ATTENTION_ARGS_V1));
    if (a.dtype != BV_F16 && a.dtype != BV_BF16)
        return fail(BV_E_UNSUPPORTED, "attention: dtype %u is not BV_F16 or BV_BF16", a.dtype);
    if (a.heads_q == 0 || a.heads_k == 0 || a.heads_q % a.heads_k)
        return fail(BV_E_INVALID, "attention: heads_q %u is no multiple of heads_k %u", a.heads_q, a.heads_k);
    if (a.heads_q > 32768) return fail(BV_E_UNSUPPORTED, "attention: %u heads, at most 32768", a.heads_q);
    if (a.head_dim == 0) return fail(BV_E_INVALID, "attention: head_dim is 0");
    if (a.head_dim > 256) return fail(BV_E_UNSUPPORTED, "attention: head_dim %u exceeds 256", a.head_dim);
    if (a.tokens_q > TOKENS_MOST || a.tokens_k > TOKENS_MOST || a.batch > TOKENS_MOST)
        return fail(BV_E_INVALID, "attention: tokens and batch are at most 2^31 - 1");
    // tiles that hold a sequence's last rows and keys end past them, in 32 bits
    if (a.tokens_k > TOKENS_MOST - 1024)
        return fail(BV_E_UNSUPPORTED, "attention: %llu keys, at most 2^31 - 1025", (unsigned long long)a.tokens_k);
    if (a.tokens_q * (a.heads_q / a.heads_k) > TOKENS_MOST - 1024)
        return fail(BV_E_UNSUPPORTED, "attention: %llu queries of %u heads a key head, at most 2^31 - 1025 in all",
                    (unsigned long long)a.tokens_q, a.heads_q / a.heads_k);
    if (!std::isfinite(a.scale)) return fail(BV_E_INVALID, "attention: scale is not finite");
    Span q{"q"}, k{"k"}, v{"v"}, o{"o"}, cq{"cu_q"}, ck{"cu_k"};
    OK_OR_RETURN(check_heads("attention", q, a.q, a.tokens_q, a.heads_q, a.head_dim, a.q_stride, a.q_head_stride, 2));
    OK_OR_RETURN(check_heads("attention", o, a.o, a.tokens_q, a.heads_q, a.head_dim, a.o_stride, a.o_head_stride, 2));
    OK_OR_RETURN(check_heads("attention", k, a.k, a.tokens_k, a.heads_k, a.head_dim, a.k_stride, a.k_head_stride, 2));
    OK_OR_RETURN(check_heads("attention", v, a.v, a.tokens_k, a.heads_k, a.head_dim, a.v_stride, a.v_head_stride, 2));
    uint64_t one = 0;
    OK_OR_RETURN(check_matrix("attention", cq, a.cu_q, (uint64_t)a.batch + 1, 1, one, 4));
    one = 0;
    OK_OR_RETURN(check_matrix("attention", ck, a.cu_k, (uint64_t)a.batch + 1, 1, one, 4));
    OK_OR_RETURN(check_apart("attention", o, {q, k, v, cq, ck}));
    std::lock_guard<std::mutex> lock(e->mu);
    OK_OR_RETURN(embed_live(e));
    if (a.batch == 0 || a.tokens_q == 0) return BV_OK;
    AttentionArgs t{};
    t.dtype = (int)a.dtype;
    t.causal = a.causal != 0;
    t.hq = a.heads_q;
    t.hk = a.heads_k;
    t.d = a.head_dim;
    t.batch = a.batch;
    t.max_q = a.max_q;
    t.max_k = a.max_k;
    t.scale = a.scale != 0 ? a.scale : (float)(1.0 / std::sqrt((double)a.head_dim));
    t.tq = a.tokens_q;
    t.tk = a.tokens_k;
    t.q = a.q;
    t.k = a.k;
    t.v = a.v;
    t.o = a.o;
    t.cu_q = a.cu_q;
    t.cu_k = a.cu_k;
    t.sq = a.q_stride;
    t.sqh = a.q_head_stride;
    t.sk = a.k_stride;
    t.skh = a.k_head_stride;
    t.sv = a.v_stride;
    t.svh = a.v_head_stride;
    t.so = a.o_stride;
    t.soh = a.o_head_stride;
    t.zeros = e->zeros;
    if (a.window) {
        t.left = std::min(a.window_left, 0x7fffffffu);
        t.right = std::min(a.window_right, 0x7fffffffu);
        t.sinks = std::min(a.sinks, 0x7fffffffu);
        // a window that ends nowhere hides nothing
        t.local = t.left < a.tokens_k || (!t.causal && t.right < std::max(a.tokens_q, a.tokens_k));
    }
    void *ws = nullptr;
    OK_OR_RETURN(embed_workspace(e, attention_workspace(t), &ws));
    HIPX(e->dev, launch_attention(t, ws, e->stream), "attention kernel");
    return BV_OK;
}

// ----------------------------------------------------------- norm, pooling --
extern "C" int bv_embed_norm(bv_embed *e, const bv_embed_norm_args *args) {
    bv_embed_norm_args a;
    OK_OR_RETURN(check_args(e, args, a, "norm"));
    if (a.dtype > BV_BF16 || a.out_dtype > BV_BF16 || ((a.weight || a.bias) && a.weight_dtype > BV_BF16))
        return fail(BV_E_UNSUPPORTED, "norm: unknown dtype");
    if (a.norm > BV_NORM_RMS) return fail(BV_E_INVALID, "norm: unknown norm %u", a.norm);
    if (a.pool > BV_POOL_LAST) return fail(BV_E_INVALID, "norm: unknown pooling %u", a.pool);
    if (a.pool && a.out_dtype != BV_F32) return fail(BV_E_UNSUPPORTED, "norm: pooled rows are BV_F32");
    if (a.dim == 0) return fail(BV_E_INVALID, "norm: dim is 0");
    if (a.dim > NORM_MAX_DIM) return fail(BV_E_UNSUPPORTED, "norm: dim %u exceeds %u", a.dim, NORM_MAX_DIM);
    if (a.norm && !(a.eps >= 0)) return fail(BV_E_INVALID, "norm: eps is negative");
    if (a.pool && (a.tokens > TOKENS_MOST || a.batch > TOKENS_MOST))
        return fail(BV_E_INVALID, "norm: pooled tokens and batch are at most 2^31 - 1");
    const uint64_t in = size_of(a.dtype), out = size_of(a.out_dtype), wt = size_of(a.weight_dtype);
    Span x{"x"}, w{"weight"}, b{"bias"}, c{"cu"}, y{"y"};
    OK_OR_RETURN(check_matrix("norm", x, a.x, a.tokens, a.dim, a.x_stride, in));
    OK_OR_RETURN(check_matrix("norm", y, a.y, a.pool ? a.batch : a.tokens, a.dim, a.y_stride, out));
    uint64_t one = 0;
    if (a.weight) OK_OR_RETURN(check_matrix("norm", w, a.weight, 1, a.dim, one, wt));
    one = 0;
    if (a.bias) OK_OR_RETURN(check_matrix("norm", b, a.bias, 1, a.dim, one, wt));
    one = 0;
    if (a.pool) OK_OR_RETURN(check_matrix("norm", c, a.cu, (uint64_t)a.batch + 1, 1, one, 4));
    const bool in_place = !a.pool && a.x == a.y && a.x_stride == a.y_stride && a.dtype == a.out_dtype;
    if (!in_place) OK_OR_RETURN(check_apart("norm", y, {x}));
    OK_OR_RETURN(check_apart("norm", y, {w, b, c}));
    std::lock_guard<std::mutex> lock(e->mu);
    OK_OR_RETURN(embed_live(e));
    if (a.pool ? a.batch == 0 : a.tokens == 0) return BV_OK;
    NormArgs n{};
    n.dtype = (int)a.dtype;
    n.out_dtype = (int)a.out_dtype;
    n.wtype = (int)a.weight_dtype;
    n.norm = (int)a.norm;
    n.pool = (int)a.pool;
    n.unit = a.unit != 0;
    n.batch = a.batch;
    n.dim = a.dim;
    n.eps = a.eps;
    n.tokens = a.tokens;
    n.x = a.x;
    n.w = a.weight;
    n.b = a.bias;
    n.cu = a.cu;
    n.y = a.y;
    n.ldx = a.x_stride;
    n.ldy = a.y_stride;
    if (n.pool == BV_POOL_MEAN) {
        void *ws;
        OK_OR_RETURN(embed_workspace(e, (size_t)pool_chunks(n.tokens, n.batch) * n.dim * 4, &ws));
        n.part = (float *)ws;
    }
    HIPX(e->dev, launch_norm(n, e->stream), "norm kernel");
    return BV_OK;
}

extern "C" int bv_embed_add_norm(bv_embed *e, const bv_embed_add_norm_args *args) {
    bv_embed_add_norm_args a;
    OK_OR_RETURN(check_args(e, args, a, "add_norm"));
    if (a.dtype > BV_BF16 || a.out_dtype > BV_I8 || ((a.weight || a.bias) && a.weight_dtype > BV_BF16))
        return fail(BV_E_UNSUPPORTED, "add_norm: unknown dtype");
    if (a.residual && a.residual_dtype != a.dtype && a.residual_dtype != BV_F32)
        return fail(BV_E_UNSUPPORTED, "add_norm: residual_dtype %u is neither dtype nor BV_F32", a.residual_dtype);
    if (a.norm > BV_NORM_RMS) return fail(BV_E_INVALID, "add_norm: unknown norm %u", a.norm);
    if (a.dim == 0) return fail(BV_E_INVALID, "add_norm: dim is 0");
    if (a.dim > NORM_MAX_DIM) return fail(BV_E_UNSUPPORTED, "add_norm: dim %u exceeds %u", a.dim, NORM_MAX_DIM);
    if (a.norm && !(a.eps >= 0)) return fail(BV_E_INVALID, "add_norm: eps is negative");
    if (a.total && !a.residual) return fail(BV_E_INVALID, "add_norm: total without a residual");
    const bool codes = a.out_dtype == BV_I8;
    const uint64_t in = size_of(a.dtype), added = size_of(a.residual_dtype), out = size_of(a.out_dtype), wt = size_of(a.weight_dtype);
    Span x{"x"}, r{"residual"}, w{"weight"}, b{"bias"}, t{"total"}, y{"y"}, sc{"scales"};
    OK_OR_RETURN(check_matrix("add_norm", x, a.x, a.tokens, a.dim, a.x_stride, in));
    OK_OR_RETURN(check_matrix("add_norm", y, a.y, a.tokens, a.dim, a.y_stride, out));
    if (a.residual) OK_OR_RETURN(check_matrix("add_norm", r, a.residual, a.tokens, a.dim, a.residual_stride, added));
    if (a.total) OK_OR_RETURN(check_matrix("add_norm", t, a.total, a.tokens, a.dim, a.total_stride, added));
    uint64_t one = 0;
    if (a.weight) OK_OR_RETURN(check_matrix("add_norm", w, a.weight, 1, a.dim, one, wt));
    one = 0;
    if (a.bias) OK_OR_RETURN(check_matrix("add_norm", b, a.bias, 1, a.dim, one, wt));
    one = 0;
    if (codes) OK_OR_RETURN(check_matrix("add_norm", sc, a.scales, 1, a.tokens, one, 4));
    const bool y_is_x = a.x == a.y && a.x_stride == a.y_stride && a.dtype == a.out_dtype;
    const bool t_is_x = a.total == a.x && a.total_stride == a.x_stride && a.residual_dtype == a.dtype;
    const bool t_is_r = a.total == a.residual && a.total_stride == a.residual_stride;
    if (!y_is_x) OK_OR_RETURN(check_apart("add_norm", y, {x}));
    OK_OR_RETURN(check_apart("add_norm", y, {r, w, b, t, sc}));
    if (!t_is_x) OK_OR_RETURN(check_apart("add_norm", t, {x}));
    if (!t_is_r) OK_OR_RETURN(check_apart("add_norm", t, {r}));
    OK_OR_RETURN(check_apart("add_norm", t, {w, b, sc}));
    OK_OR_RETURN(check_apart("add_norm", sc, {x, r, w, b}));
    std::lock_guard<std::mutex> lock(e->mu);
    OK_OR_RETURN(embed_live(e));
    if (a.tokens == 0) return BV_OK;
    AddNormArgs n{};
    n.dtype = (int)a.dtype;
    n.r_dtype = (int)a.residual_dtype;
    n.out_dtype = (int)a.out_dtype;
    n.wtype = (int)a.weight_dtype;
    n.norm = (int)a.norm;
    n.dim = a.dim;
    n.eps = a.eps;
    n.tokens = a.tokens;
    n.x = a.x;
    n.r = a.residual;
    n.w = a.weight;
    n.b = a.bias;
    n.total = a.total;
    n.y = a.y;
    n.scales = (float *)a.scales;
    n.ldx = a.x_stride;
    n.ldr = a.residual_stride;
    n.ldt = a.total_stride;
    n.ldy = a.y_stride;
    HIPX(e->dev, launch_add_norm(n, e->stream), "add_norm kernel");
    return BV_OK;
}
