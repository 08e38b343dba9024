// The C entry points of libdgnn_ops.so (include/dgnn_ops.h): argument checks, the device, the launch.
#include "ops.h"

#include <cmath>

namespace {

thread_local int g_last_hip_error = 0;

int hip_failed(hipError_t err)
{
    g_last_hip_error = (int)err;
    (void)hipGetLastError();            // the runtime keeps it as well, for whoever asks next: it has been told here
    return DGNN_HIP_ERROR;
}

// The caller's current device is what it was when a call returns.
class DeviceGuard {
public:
    explicit DeviceGuard(int device)
    {
        error_ = hipGetDevice(&previous_);
        if (error_ == hipSuccess && previous_ != device) {
            error_ = hipSetDevice(device);
            changed_ = error_ == hipSuccess;
        }
    }
    ~DeviceGuard()
    {
        if (changed_) (void)hipSetDevice(previous_);
    }
    hipError_t error() const { return error_; }

private:
    int previous_ = 0;
    bool changed_ = false;
    hipError_t error_ = hipSuccess;
};

constexpr int64_t kMaxExtent = INT32_MAX;

bool extent_ok(int64_t v) { return v >= 0 && v <= kMaxExtent; }
// `count` rows at this stride: their offsets in bytes stay far inside 64 bits
bool stride_ok(int64_t stride, int64_t count) { return stride >= 0 && stride <= ((int64_t)1 << 56) / (count > 1 ? count : 1); }
int64_t size_of(int32_t type)
{
    switch (type) {
    case DGNN_F16: case DGNN_BF16: return 2;
    case DGNN_I64: return 8;
    default: return 4;
    }
}
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }
bool float_type(int32_t t) { return t == DGNN_F16 || t == DGNN_BF16 || t == DGNN_F32; }
bool activation_ok(int32_t a) { return a >= DGNN_ACT_IDENTITY && a <= DGNN_ACT_SILU; }

bool holds(const void* workspace, int64_t bytes, int64_t need) { return need == 0 || (workspace && bytes >= need && aligned(workspace, 256)); }

// rows of `width` bytes, `pitch` bytes apart
struct Rows {
    const void* data;
    int64_t rows, pitch, width;
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(data); }
    uintptr_t end() const { return begin() + (uintptr_t)((rows - 1) * pitch + width); }
};

// Whether two sets of rows may share a byte.  Two column ranges of one buffer (equal pitch) are told apart; otherwise overlapping spans count.
bool may_overlap(const Rows& a, const Rows& b)
{
    if (!a.data || !b.data || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
    if (a.end() <= b.begin() || b.end() <= a.begin()) return false;
    const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
    if ((a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) || pitch < a.width || pitch < b.width) return true;
    const int64_t off = (int64_t)((a.begin() < b.begin() ? b.begin() - a.begin() : (uintptr_t)pitch - (a.begin() - b.begin()) % (uintptr_t)pitch) % (uintptr_t)pitch);
    return off < a.width || off + b.width > pitch;      // b's columns begin `off` bytes behind a's, cyclically
}

// An output that is allowed to BE an input (`same`) but not to overlap it otherwise.
bool bad_alias(const Rows& out, const Rows& in)
{
    if (out.data == in.data && out.width == in.width && (out.rows <= 1 || out.pitch == in.pitch)) return false;
    return may_overlap(out, in);
}

int check(const dgnn_dense_args* a)
{
    if (!a || !extent_ok(a->m) || !extent_ok(a->n) || !extent_ok(a->k)) return DGNN_BAD_ARGUMENT;
    if (!stride_ok(a->ldx, a->m) || !stride_ok(a->ldw, a->n) || !stride_ok(a->ldz, a->m) || !stride_ok(a->ldy, a->m)) return DGNN_BAD_ARGUMENT;
    if (!activation_ok(a->activation) || !float_type(a->type) || !float_type(a->out_type) || !float_type(a->bias_type)) return DGNN_BAD_ARGUMENT;
    if (a->type == DGNN_F32) return DGNN_UNSUPPORTED;
    if (a->out_type != a->type && a->out_type != DGNN_F32) return DGNN_UNSUPPORTED;
    if (a->bias_type != a->type && a->bias_type != DGNN_F32) return DGNN_UNSUPPORTED;
    if (a->m == 0 || a->n == 0) return DGNN_OK;
    if (!a->y || (a->k > 0 && (!a->x || !a->w))) return DGNN_BAD_ARGUMENT;
    if (a->m > 1 && a->ldy < a->n) return DGNN_BAD_ARGUMENT;
    const int64_t e = size_of(a->type), o = size_of(a->out_type);
    if (!aligned(a->x, e) || !aligned(a->w, e) || !aligned(a->bias, size_of(a->bias_type)) || !aligned(a->z, o) || !aligned(a->y, o)) return DGNN_BAD_ARGUMENT;
    const Rows y{a->y, a->m, a->ldy * o, a->n * o};
    if (a->k > 0 && (may_overlap(y, {a->x, a->m, a->ldx * e, a->k * e}) || may_overlap(y, {a->w, a->n, a->ldw * e, a->k * e}))) return DGNN_BAD_ARGUMENT;
    if (a->z && bad_alias(y, {a->z, a->m, a->ldz * o, a->n * o})) return DGNN_BAD_ARGUMENT;
    if (may_overlap(y, {a->bias, 1, 0, a->n * size_of(a->bias_type)})) return DGNN_BAD_ARGUMENT;
    return DGNN_OK;
}

// Whether [n][p][c] with these strides can be written: distinct elements at distinct places.
bool writable(int64_t n, int64_t p, int64_t c, int64_t sn, int64_t sp)
{
    if (p > 1 && sp < c) return false;
    return n <= 1 || sn >= (p - 1) * sp + c;
}

int check(const dgnn_group_norm_args* a)
{
    if (!a || !extent_ok(a->n) || !extent_ok(a->p) || !extent_ok(a->c) || a->groups < 1 || a->groups > kMaxExtent) return DGNN_BAD_ARGUMENT;
    for (int64_t stride : {a->x_n, a->z_n, a->y_n})
        if (!stride_ok(stride, a->n)) return DGNN_BAD_ARGUMENT;
    for (int64_t stride : {a->x_p, a->z_p, a->y_p})
        if (!stride_ok(stride, a->p)) return DGNN_BAD_ARGUMENT;
    if (a->c % a->groups != 0 || !(a->eps >= 0.0f) || std::isinf(a->eps)) return DGNN_BAD_ARGUMENT;
    if (!activation_ok(a->activation) || !float_type(a->type) || !float_type(a->affine_type)) return DGNN_BAD_ARGUMENT;
    if (a->affine_type != a->type && a->affine_type != DGNN_F32) return DGNN_UNSUPPORTED;
    if (a->n == 0 || a->p == 0 || a->c == 0) return DGNN_OK;
    if (a->p > kMaxExtent / a->c * 64) return DGNN_UNSUPPORTED;         // one sample: at most 2^37 elements
    if (!a->x || !a->y || !writable(a->n, a->p, a->c, a->y_n, a->y_p)) return DGNN_BAD_ARGUMENT;
    const int64_t e = size_of(a->type), f = size_of(a->affine_type);
    if (!aligned(a->x, e) || !aligned(a->z, e) || !aligned(a->y, e) || !aligned(a->weight, f) || !aligned(a->bias, f)) return DGNN_BAD_ARGUMENT;
    // As rows of whole samples: y is exactly x (or z), or shares nothing with it.
    const auto span = [&](const void* p, int64_t sn, int64_t sp) { return Rows{p, a->n, sn * e, ((a->p - 1) * sp + a->c) * e}; };
    const auto alias = [&](const void* p, int64_t sn, int64_t sp) {
        if (p == a->y && (a->n == 1 || sn == a->y_n) && (a->p == 1 || sp == a->y_p)) return false;
        // positions of equal stride in both are told apart by their columns, also across samples that follow on each other
        const Rows ry{a->y, a->n == 1 ? a->p : (a->y_n == a->p * a->y_p ? a->n * a->p : 0), a->y_p * e, a->c * e};
        const Rows rp{p, a->n == 1 ? a->p : (sn == a->p * sp ? a->n * a->p : 0), sp * e, a->c * e};
        if (ry.rows > 0 && rp.rows > 0) return may_overlap(ry, rp);
        return may_overlap(span(a->y, a->y_n, a->y_p), span(p, sn, sp));
    };
    if (alias(a->x, a->x_n, a->x_p) || (a->z && alias(a->z, a->z_n, a->z_p))) return DGNN_BAD_ARGUMENT;
    const Rows y = span(a->y, a->y_n, a->y_p);
    if (may_overlap(y, {a->weight, 1, 0, a->c * f}) || may_overlap(y, {a->bias, 1, 0, a->c * f})) return DGNN_BAD_ARGUMENT;
    return DGNN_OK;
}

int check(const dgnn_logits_args* a)
{
    if (!a || !extent_ok(a->b) || !extent_ok(a->v) || !extent_ok(a->t)) return DGNN_BAD_ARGUMENT;
    for (int64_t stride : {a->ld_logits, a->ld_out, a->ld_mask, a->ld_bias, a->ld_history})
        if (!stride_ok(stride, a->b)) return DGNN_BAD_ARGUMENT;
    if (!float_type(a->type) || !float_type(a->out_type) || !float_type(a->bias_type)) return DGNN_BAD_ARGUMENT;
    if (a->history_type != DGNN_I32 && a->history_type != DGNN_I64) return DGNN_BAD_ARGUMENT;
    if (a->out_type != a->type && a->out_type != DGNN_F32) return DGNN_UNSUPPORTED;
    if (a->bias_type != a->type && a->bias_type != DGNN_F32) return DGNN_UNSUPPORTED;
    if (!a->repetition && !(a->repetition_all > 0.0f && std::isfinite(a->repetition_all))) return DGNN_BAD_ARGUMENT;
    if ((!a->presence && !std::isfinite(a->presence_all)) || (!a->frequency && !std::isfinite(a->frequency_all))) return DGNN_BAD_ARGUMENT;
    if (a->b == 0 || a->v == 0) return DGNN_OK;
    if (!a->logits || !a->out) return DGNN_BAD_ARGUMENT;
    const int64_t words = (a->v + 31) / 32;
    if (a->b > 1 && a->ld_out < a->v) return DGNN_BAD_ARGUMENT;
    const int64_t e = size_of(a->type), o = size_of(a->out_type), f = size_of(a->bias_type);
    if (!aligned(a->logits, e) || !aligned(a->out, o) || !aligned(a->mask, 4) || !aligned(a->bias, f)) return DGNN_BAD_ARGUMENT;
    if (!aligned(a->history, size_of(a->history_type)) || !aligned(a->lengths, 4) || !aligned(a->prompt_lengths, 4)) return DGNN_BAD_ARGUMENT;
    if (!aligned(a->repetition, 4) || !aligned(a->presence, 4) || !aligned(a->frequency, 4)) return DGNN_BAD_ARGUMENT;
    const Rows out{a->out, a->b, a->ld_out * o, a->v * o};
    if (bad_alias(out, {a->logits, a->b, a->ld_logits * e, a->v * e})) return DGNN_BAD_ARGUMENT;
    if (may_overlap(out, {a->mask, a->b, a->ld_mask * 4, words * 4}) || may_overlap(out, {a->bias, a->b, a->ld_bias * f, a->v * f})) return DGNN_BAD_ARGUMENT;
    if (may_overlap(out, {a->history, a->b, a->ld_history * size_of(a->history_type), a->t * size_of(a->history_type)})) return DGNN_BAD_ARGUMENT;
    for (const void* p : {(const void*)a->lengths, (const void*)a->prompt_lengths, (const void*)a->repetition, (const void*)a->presence, (const void*)a->frequency})
        if (may_overlap(out, {p, 1, 0, a->b * 4})) return DGNN_BAD_ARGUMENT;
    return DGNN_OK;
}

template <typename Args, typename Launch>
int run(int device, void* stream, const Args& args, Launch launch)
{
    if (device < 0) return DGNN_BAD_ARGUMENT;
    const DeviceGuard guard(device);
    if (guard.error() != hipSuccess) return hip_failed(guard.error());
    const hipError_t err = launch(args, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? DGNN_OK : hip_failed(err);
}

}  // namespace

extern "C" {

__attribute__((visibility("default"))) int dgnn_ops_last_hip_error(void) { return g_last_hip_error; }

__attribute__((visibility("default"))) int dgnn_dense_workspace(const dgnn_dense_args* args, int64_t* bytes)
{
    if (!bytes) return DGNN_BAD_ARGUMENT;
    *bytes = 0;
    const int status = check(args);
    if (status != DGNN_OK || args->m == 0 || args->n == 0) return status;
    *bytes = dgnn::ops::dense_workspace(*args);
    return DGNN_OK;
}

__attribute__((visibility("default"))) int dgnn_dense(int device, void* hip_stream, const dgnn_dense_args* args)
{
    const int status = check(args);
    if (status != DGNN_OK || args->m == 0 || args->n == 0) return status;
    if (!holds(args->workspace, args->workspace_bytes, dgnn::ops::dense_workspace(*args))) return DGNN_BAD_ARGUMENT;
    return run(device, hip_stream, *args, dgnn::ops::launch_dense);
}

__attribute__((visibility("default"))) int dgnn_group_norm_workspace(const dgnn_group_norm_args* args, int64_t* bytes)
{
    if (!bytes) return DGNN_BAD_ARGUMENT;
    *bytes = 0;
    const int status = check(args);
    if (status != DGNN_OK || args->n == 0 || args->p == 0 || args->c == 0) return status;
    *bytes = dgnn::ops::group_norm_workspace(*args);
    return DGNN_OK;
}

__attribute__((visibility("default"))) int dgnn_group_norm(int device, void* hip_stream, const dgnn_group_norm_args* args)
{
    const int status = check(args);
    if (status != DGNN_OK || args->n == 0 || args->p == 0 || args->c == 0) return status;
    if (!holds(args->workspace, args->workspace_bytes, dgnn::ops::group_norm_workspace(*args))) return DGNN_BAD_ARGUMENT;
    return run(device, hip_stream, *args, dgnn::ops::launch_group_norm);
}

__attribute__((visibility("default"))) int dgnn_adjust_logits(int device, void* hip_stream, const dgnn_logits_args* args)
{
    const int status = check(args);
    if (status != DGNN_OK || args->b == 0 || args->v == 0) return status;
    return run(device, hip_stream, *args, dgnn::ops::launch_adjust_logits);
}

}  // extern "C"
