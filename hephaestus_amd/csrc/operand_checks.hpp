// Checks of the operands of layer and training operators, made before anything
// is launched, and the plans that bind them.  Host code.
#pragma once

#include "hx_internal.hpp"

#include <cstdlib>
#include <new>

namespace hx {

inline hx_status check_layer_dtype(hx_dtype d, uint32_t *size) {
    if (d != HX_DTYPE_F32 && d != HX_DTYPE_BF16)
        return fail(HX_ERR_INVALID_CONFIGURATION, "layer operators take f32 or bf16 operands, got dtype %d", (int)d);
    *size = d == HX_DTYPE_F32 ? 4 : 2;
    return HX_OK;
}

// The bytes that a view reaches lie in [first, end): from first on, `run` bytes at
// each sum of whole steps.  Empty views reach none.
struct Span {
    uintptr_t first = 0, end = 0;
    const void *base = nullptr;
    const hx_layout *layout = nullptr;
    uint64_t run = 0;
    uint32_t steps = 0;
    uint64_t step[HX_MAX_RANK] = {}, count[HX_MAX_RANK] = {};
};

// Whether Σ step·x = target has a solution with each x in [0, most], by trying
// the values of x that the smaller steps can complete, the largest step first.
// Where each step passes what the smaller ones reach together, as in views of
// rows within rows, those are a few; a search that grows beyond `kTries` is given
// up and counts as a solution.
class StepSums {
  public:
    void add(uint64_t step, uint64_t most) {
        if (step == 0 || most == 0) return;
        uint32_t at = 0;
        while (at < n_ && step_[at] > step) ++at;
        if (at < n_ && step_[at] == step) {
            most_[at] += most;
            return;
        }
        for (uint32_t i = n_++; i > at; --i) step_[i] = step_[i - 1], most_[i] = most_[i - 1];
        step_[at] = step;
        most_[at] = most;
    }
    bool reach(__int128 target) {
        __int128 sum = 0;
        reach_[n_] = 0;
        for (uint32_t i = n_; i-- > 0;) reach_[i] = sum += (__int128)step_[i] * most_[i];
        tries_ = 0;
        return from(0, target);
    }

  private:
    static constexpr uint32_t kMost = 2 * HX_MAX_RANK + 1, kTries = 1 << 14;
    uint32_t n_ = 0, tries_ = 0;
    uint64_t step_[kMost], most_[kMost];
    __int128 reach_[kMost + 1];

    bool from(uint32_t i, __int128 target) {
        if (target < 0 || target > reach_[i]) return false;
        if (target == 0) return true;
        if (++tries_ > kTries) return true;
        const __int128 step = step_[i], rest = target - reach_[i + 1];
        const __int128 low = rest > 0 ? (rest + step - 1) / step : 0, high = target / step;
        for (__int128 x = low; x <= high && x <= most_[i]; ++x)
            if (from(i + 1, target - x * step)) return true;
        return false;
    }
};

// Whether two views share a byte: a.first + Σ a's steps + a byte of the run meets
// the same of b.  With b's steps counted from their ends all of them add up.
inline bool overlap(const Span &a, const Span &b) {
    if (a.first >= b.end || b.first >= a.end) return false;
    StepSums sums;
    for (uint32_t i = 0; i < a.steps; ++i) sums.add(a.step[i], a.count[i] - 1);
    for (uint32_t i = 0; i < b.steps; ++i) sums.add(b.step[i], b.count[i] - 1);
    sums.add(1, a.run - 1 + (b.run - 1));
    return sums.reach((__int128)b.end - 1 - (__int128)a.first);
}

// The same elements at the same indices.
inline bool same_view(const Span &a, const Span &b) {
    if (a.base != b.base || a.layout->offset != b.layout->offset) return false;
    for (uint32_t d = 0; d < a.layout->rank; ++d)
        if (a.layout->shape[d] > 1 && a.layout->strides[d] != b.layout->strides[d]) return false;
    return true;
}

// Distinct indices reach distinct elements: no two differ by a whole number y of
// steps in each dimension that come to nothing, Σ stride·y = 0.  With d the first
// dimension of y ≠ 0, y_d is taken as 1 on and the later ones from 1 - shape on.
inline bool is_injective(const hx_layout &l) {
    for (uint32_t d = 0; d < l.rank; ++d) {
        if (l.shape[d] <= 1) continue;
        const uint64_t step = (uint64_t)std::llabs(l.strides[d]);
        if (step == 0) return false;
        StepSums sums;
        __int128 target = -(__int128)step;
        sums.add(step, l.shape[d] - 2);
        for (uint32_t e = d + 1; e < l.rank; ++e) {
            if (l.shape[e] <= 1) continue;
            const uint64_t other = (uint64_t)std::llabs(l.strides[e]);
            sums.add(other, 2 * (l.shape[e] - 1));
            target += (__int128)other * (l.shape[e] - 1);
        }
        if (sums.reach(target)) return false;
    }
    return true;
}

// One operand: its rank and shape, its buffer, its contiguous last dimension.
inline hx_status check_view(const void *buf, uint64_t buf_len, const hx_layout *l, uint32_t rank, const uint64_t *shape,
                     uint32_t size, bool written, const char *what, Span *span) {
    HX_TRY(layout_basic_check(l, what));
    if (l->rank != rank)
        return fail(HX_ERR_DISPATCH_FAILED, "%s needs a rank-%u view, got rank %u", what, rank, l->rank);
    for (uint32_t d = 0; d < rank; ++d)
        if (l->shape[d] != shape[d]) {
            hx_layout want{};
            want.rank = rank;
            for (uint32_t i = 0; i < rank; ++i) want.shape[i] = shape[i];
            return fail(HX_ERR_DISPATCH_FAILED, "%s has shape %s, expected %s", what, shape_string(*l).c_str(),
                        shape_string(want).c_str());
        }
    uint64_t n = 0;
    HX_TRY(hx_layout_checked_size(l, &n));
    *span = Span{};
    span->base = buf;
    span->layout = l;
    if (n == 0) return HX_OK;
    HX_TRY(hx_layout_validate_storage_len(l, buf_len));
    if (!buf) return fail(HX_ERR_DISPATCH_FAILED, "%s buffer is null", what);
    if ((uintptr_t)buf % size) return fail(HX_ERR_DISPATCH_FAILED, "%s is not aligned to its elements", what);
    if (l->shape[rank - 1] > 1 && l->strides[rank - 1] != 1)
        return fail(HX_ERR_DISPATCH_FAILED, "%s needs a contiguous last dimension, got stride %lld", what,
                    (long long)l->strides[rank - 1]);
    if (written && !is_injective(*l))
        return fail(HX_ERR_DISPATCH_FAILED, "%s layout must not reach an element twice", what);
    int64_t lo = (int64_t)l->offset, hi = lo; // within the buffer, as just validated
    for (uint32_t d = 0; d < rank; ++d) {
        const int64_t reach = (int64_t)(l->shape[d] - 1) * l->strides[d];
        if (reach < 0) lo += reach;
        else hi += reach;
    }
    span->first = (uintptr_t)buf + (uint64_t)lo * size;
    span->end = (uintptr_t)buf + ((uint64_t)hi + 1) * size;
    span->run = l->shape[rank - 1] * size;
    for (uint32_t d = 0; d + 1 < rank; ++d) {
        span->step[span->steps] = (uint64_t)std::llabs(l->strides[d]) * size;
        span->count[span->steps++] = l->shape[d];
    }
    return HX_OK;
}

// An operand that may be left out is so by its layout; a buffer without one is
// not what its caller means.
inline hx_status check_left_out(const void *buf, uint64_t buf_len, const hx_layout *l, const char *what) {
    if (!l && (buf || buf_len))
        return fail(HX_ERR_INVALID_CONFIGURATION, "%s has a buffer and no layout", what);
    return HX_OK;
}

// A whole buffer of `len` elements where `want` are expected.
inline hx_status check_vector(const void *buf, uint64_t len, uint64_t want, uint32_t size, const char *what, Span *span) {
    if (len != want) return length_mismatch(want, len);
    *span = Span{};
    span->base = buf;
    if (want == 0) return HX_OK;
    if (!buf) return fail(HX_ERR_DISPATCH_FAILED, "%s buffer is null", what);
    if ((uintptr_t)buf % size) return fail(HX_ERR_DISPATCH_FAILED, "%s is not aligned to its elements", what);
    span->first = (uintptr_t)buf;
    span->end = span->first + want * size;
    span->run = want * size;
    return HX_OK;
}

inline hx_status check_apart(const Span &out, const char *out_name, const Span &other, const char *other_name) {
    if (overlap(out, other))
        return fail(HX_ERR_DISPATCH_FAILED, "%s must not overlap %s", out_name, other_name);
    return HX_OK;
}

template <typename T> T *at(T *buf, const hx_layout *l, uint32_t size) {
    return buf ? (T *)((uintptr_t)buf + l->offset * size) : nullptr;
}

inline int64_t stride_of(const hx_layout *l, uint32_t d) { return l->shape[d] > 1 ? l->strides[d] : 0; }

// A plan with `bytes` of workspace, which the operators write before they
// read: it is not cleared.
template <typename Plan, typename Args>
hx_status make_plan(hx_device *dev, const Args &args, uint64_t bytes, hx_plan **out) {
    HX_TRY(bind_device(dev));
    Plan *p = new (std::nothrow) Plan();
    if (!p) return fail(HX_ERR_ALLOCATION_FAILED, "host allocation of plan failed");
    p->dev = dev;
    p->args = args;
    if (bytes) {
        const hipError_t err = hipMalloc(&p->ws, bytes);
        if (err != hipSuccess) {
            p->ws = nullptr;
            delete p;
            return hip_fail(HX_ERR_ALLOCATION_FAILED, err, "workspace hipMalloc");
        }
        p->ws_bytes = bytes;
    }
    *out = p;
    return ok();
}

} // namespace hx
