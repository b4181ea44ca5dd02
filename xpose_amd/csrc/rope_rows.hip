// Rotary positions of packed rows: x0' = m (x0 cos - x1 sin), x1' = m (x1 cos +
// x0 sin), the angle pos f_i of pair i.
//
// Angles. f_i in turns a position is a 64-bit fixed-point fraction, so that
// pos f_i modulo one turn is one integer product modulo 2^64, off by pos times the
// fraction's own 2^-55 at most (in fp32 the product alone is off by a thousandth of a
// turn at position 10^5). Its high word, signed, is the
// fraction of a turn in [-1/2, 1/2) that sincospif takes.
//
// Bytes bound it. A workgroup's few tokens share their cosines and sines, and a lane takes
// 16 bytes at a time: 8192 tokens of 40 heads of 128 in bf16 (168 MB) 35.3 us, 4.75 TB/s, what a
// copy reaches. 16 tokens take 3.1 us of the device and 5.0 of the host.
#include <algorithm>
#include <cmath>

#include "xp_elem.hpp"
#include "xp_launch.hpp"

namespace xp {
namespace {

constexpr uint32_t kRopeThreads = 256;

struct RopeTurns {
    uint64_t f[kMaxHeadDim / 2];    // turns a position, 2^-64 each
};
struct RopeRows {
    const void *q, *k;
    void *     q_out, *k_out;
    uint64_t   q_stride, k_stride, q_out_stride, k_out_stride;   // elements
    const int32_t* positions;
    uint32_t   n_tokens, head_dim, rot, q_heads, heads, per_block;
    float      magnitude;
};

// A workgroup turns per_block tokens: it forms their cosines and sines once
// in LDS, for all heads. An item is V pairs of one head (V elements of each
// half, or 2 V interleaved ones) or V elements behind the turned dims.
template <int ELEM, bool HALF, int V>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeRows a, RopeTurns turns) {
    extern __shared__ float2 cs[];                    // [per_block][rot / 2]
    const uint32_t pairs = a.rot / 2;
    const uint32_t t0 = blockIdx.x * a.per_block, nt = min(a.per_block, a.n_tokens - t0);
    for (uint32_t i = threadIdx.x; i < nt * pairs; i += kRopeThreads) {
        const uint32_t t = i / pairs, p = i - t * pairs;
        const uint64_t angle = uint64_t(int64_t(a.positions[t0 + t])) * turns.f[p];
        float s, c;
        sincospif(float(int32_t(angle >> 32)) * 0x1p-31f, &s, &c);
        cs[i] = {c * a.magnitude, s * a.magnitude};
    }
    __syncthreads();
    const uint32_t turned = pairs / V, tail = (a.head_dim - a.rot) / V, per_head = turned + tail;
    for (uint32_t i = threadIdx.x; i < nt * a.heads * per_head; i += kRopeThreads) {
        const uint32_t row = i / per_head, e = i - row * per_head;
        const uint32_t t = row / a.heads, h = row - t * a.heads;
        const bool isq = h < a.q_heads;
        const void* in = isq ? a.q : a.k;
        void* out = isq ? a.q_out : a.k_out;
        const uint64_t hd = uint64_t(isq ? h : h - a.q_heads) * a.head_dim, tok = t0 + t;
        const uint64_t from = tok * (isq ? a.q_stride : a.k_stride) + hd, to = tok * (isq ? a.q_out_stride : a.k_out_stride) + hd;
        float x[V], y[V];
        if (e >= turned) {
            const uint32_t d = a.rot + (e - turned) * V;
            if constexpr (V == 8) {
                load8<ELEM>(in, from + d, x);
                store8<ELEM>(out, to + d, x);
            } else {
                store1<ELEM>(out, to + d, load1<ELEM>(in, from + d));
            }
            continue;
        }
        const uint32_t d0 = HALF ? e * V : 2 * e * V, d1 = HALF ? d0 + pairs : d0 + V;
        if constexpr (V == 8) {
            load8<ELEM>(in, from + d0, x);
            load8<ELEM>(in, from + d1, y);
        } else {
            x[0] = load1<ELEM>(in, from + d0);
            y[0] = load1<ELEM>(in, from + d1);
        }
        const float2* w = cs + t * pairs + e * V;
        if constexpr (HALF || V == 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 z = w[j];
                const float u = x[j], v = y[j];
                x[j] = u * z.x - v * z.y;
                y[j] = v * z.x + u * z.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 z = w[j / 2], z1 = w[(V + j) / 2];
                const float u = x[j], v = x[j + 1], u1 = y[j], v1 = y[j + 1];
                x[j] = u * z.x - v * z.y;
                x[j + 1] = v * z.x + u * z.y;
                y[j] = u1 * z1.x - v1 * z1.y;
                y[j + 1] = v1 * z1.x + u1 * z1.y;
            }
        }
        if constexpr (V == 8) {
            store8<ELEM>(out, to + d0, x);
            store8<ELEM>(out, to + d1, y);
        } else {
            store1<ELEM>(out, to + d0, x[0]);
            store1<ELEM>(out, to + d1, y[0]);
        }
    }
}

int check_spec(const char* fn, const xp_rope_spec* r) {
    if (!r) return set_error(XP_E_ARG, "%s: the rope spec is null", fn);
    if (r->rot_dim < 2 || r->rot_dim % 2 || r->rot_dim > uint32_t(kMaxHeadDim))
        return set_error(XP_E_ARG, "%s: rot_dim %u is not even and from 2 to %d", fn, r->rot_dim, kMaxHeadDim);
    if (r->layout != XP_ROPE_HALF && r->layout != XP_ROPE_INTERLEAVED)
        return set_error(XP_E_ARG, "%s: unknown layout %d", fn, r->layout);
    if (!(r->theta > 1.0f) || !std::isfinite(r->theta)) return set_error(XP_E_ARG, "%s: theta %g is not over 1", fn, double(r->theta));
    if (r->scaling < XP_ROPE_PLAIN || r->scaling > XP_ROPE_PARTS) return set_error(XP_E_ARG, "%s: unknown scaling %d", fn, r->scaling);
    if (r->scaling != XP_ROPE_PLAIN && (!(r->factor >= 1.0f) || !std::isfinite(r->factor)))
        return set_error(XP_E_ARG, "%s: factor %g is less than 1", fn, double(r->factor));
    if ((r->scaling == XP_ROPE_BANDS || r->scaling == XP_ROPE_PARTS) &&
        (!(r->original_len > 0.0f) || !std::isfinite(r->original_len) || !(r->low > 0.0f) || !(r->high > r->low) ||
         !std::isfinite(r->high)))
        return set_error(XP_E_ARG, "%s: original_len %g, low %g, high %g: 0 < original_len and 0 < low < high", fn,
                         double(r->original_len), double(r->low), double(r->high));
    if (!std::isfinite(r->magnitude) || r->magnitude < 0.0f) return set_error(XP_E_ARG, "%s: magnitude %g", fn, double(r->magnitude));
    return XP_OK;
}

// f_i of all pairs in radians a position: powers of theta^(-2 / rot_dim) by products of
// 64 bits of mantissa (off by 2^-56 after 256), which is nearly free beside a power for each (the call: 5.6 to 5.0 us of a host).
void rope_frequencies(const xp_rope_spec& r, long double* f) {
    constexpr long double two_pi = 6.283185307179586476925286766559L;
    const uint32_t pairs = r.rot_dim / 2;
    const long double n = r.rot_dim, theta = r.theta, step = std::exp(-2.0L * std::log(theta) / n);
    long double a = 0, b = 0;
    if (r.scaling == XP_ROPE_PARTS) {
        auto index = [&](long double turns) { return n * std::log(r.original_len / (two_pi * turns)) / (2.0L * std::log(theta)); };
        a = std::min(n - 1, std::max(0.0L, std::floor(index(r.high))));
        b = std::min(n - 1, std::max(0.0L, std::ceil(index(r.low))));
    }
    long double x = 1.0L;
    for (uint32_t i = 0; i < pairs; ++i, x *= step) {
        long double keep = 1.0L;
        if (r.scaling == XP_ROPE_LINEAR) keep = 0.0L;
        if (r.scaling == XP_ROPE_BANDS)
            keep = std::min(1.0L, std::max(0.0L, (r.original_len * x / two_pi - r.low) / ((long double)(r.high) - r.low)));
        if (r.scaling == XP_ROPE_PARTS) keep = 1.0L - std::min(1.0L, std::max(0.0L, (i - a) / std::max(b - a, 1e-3L)));
        f[i] = x * keep + (r.scaling == XP_ROPE_PLAIN ? 0.0L : x / r.factor * (1.0L - keep));
    }
}

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" {

int xp_rope_frequencies(const xp_rope_spec* r, double* f, uint32_t n) {
    XP_CHECK(check_spec(__func__, r));
    XP_REQUIRE(f && n == r->rot_dim / 2, "room for %u frequencies, %u are there", n, r->rot_dim / 2);
    long double x[kMaxHeadDim / 2];
    rope_frequencies(*r, x);
    for (uint32_t i = 0; i < n; ++i) f[i] = double(x[i]);
    return XP_OK;
}

int xp_rope_rows(const xp_rows* q_out, const xp_rows* q, const xp_rows* k_out, const xp_rows* k,
                 const int32_t* positions, uint32_t n_tokens, uint32_t head_dim, const xp_rope_spec* r,
                 xp_stream stream) {
    XP_CHECK(check_spec(__func__, r));
    XP_REQUIRE(head_dim % 2 == 0 && head_dim <= uint32_t(kMaxHeadDim) && r->rot_dim <= head_dim,
               "head_dim %u is not even, at most %d and at least rot_dim %u", head_dim, kMaxHeadDim, r->rot_dim);
    XP_CHECK(check_rows(__func__, "q", q, head_dim, 1));
    XP_CHECK(check_rows(__func__, "q_out", q_out, head_dim, 1));
    XP_REQUIRE(q_out->heads == q->heads && q_out->elem == q->elem, "q_out has not q's heads and elem");
    XP_REQUIRE((k != nullptr) == (k_out != nullptr), "k and k_out are both given or both NULL");
    if (k) {
        XP_CHECK(check_rows(__func__, "k", k, head_dim, 1));
        XP_CHECK(check_rows(__func__, "k_out", k_out, head_dim, 1));
        XP_REQUIRE(k_out->heads == k->heads && k_out->elem == k->elem && k->elem == q->elem,
                   "k_out has not k's heads and elem, or k not q's elem");
    }
    XP_REQUIRE(n_tokens <= 0x7FFFFFFFu, "n_tokens %u is over 2^31 - 1", n_tokens);
    if (n_tokens == 0) return XP_OK;
    XP_REQUIRE(positions, "positions is null");
    XP_CHECK(check_here(__func__, stream, q_out->data));

    RopeTurns turns;
    long double f[kMaxHeadDim / 2];
    rope_frequencies(*r, f);
    // below 2^64: f_i <= 1 radian
    for (uint32_t i = 0; i < r->rot_dim / 2; ++i) turns.f[i] = uint64_t(f[i] * (0x1p64L / 6.283185307179586476925286766559L));
    RopeRows a{q->data, k ? k->data : nullptr, q_out->data, k ? k_out->data : nullptr,
               q->stride, k ? k->stride : 0, q_out->stride, k ? k_out->stride : 0, positions,
               n_tokens, head_dim, r->rot_dim, q->heads, q->heads + (k ? k->heads : 0), 1,
               r->magnitude == 0.0f ? 1.0f : r->magnitude};
    // eight at a time where every run of eight is whole and aligned
    bool wide = r->rot_dim / 2 % 8 == 0 && (head_dim - r->rot_dim) % 8 == 0;
    for (const xp_rows* x : {q, q_out, k, k_out})
        if (x) wide = wide && reinterpret_cast<uintptr_t>(x->data) % 16 == 0 && x->stride * elem_bytes(x->elem) % 16 == 0;
    const uint32_t items = a.heads * (r->rot_dim / 2 + head_dim - r->rot_dim) / (wide ? 8 : 1);
    a.per_block = std::max(1u, std::min({kRopeThreads / std::max(items, 1u), 8u, (n_tokens + 511) / 512}));
    const dim3 grid((n_tokens + a.per_block - 1) / a.per_block);
    const size_t lds = size_t(a.per_block) * r->rot_dim / 2 * sizeof(float2);
#define XP_ROPE_V(E, H)                                                                                                    \
    if (wide) hipLaunchKernelGGL((rope_rows_kernel<E, H, 8>), grid, dim3(kRopeThreads), lds, as_stream(stream), a, turns); \
    else hipLaunchKernelGGL((rope_rows_kernel<E, H, 1>), grid, dim3(kRopeThreads), lds, as_stream(stream), a, turns);
#define XP_ROPE(E)                          \
    if (r->layout == XP_ROPE_HALF) {        \
        XP_ROPE_V(E, true)                  \
    } else {                                \
        XP_ROPE_V(E, false)                 \
    }
    if (q->elem == XP_ELEM_F32) {
        XP_ROPE(XP_ELEM_F32)
    } else if (q->elem == XP_ELEM_F16) {
        XP_ROPE(XP_ELEM_F16)
    } else {
        XP_ROPE(XP_ELEM_BF16)
    }
#undef XP_ROPE
#undef XP_ROPE_V
    XP_LAUNCHED();
    return XP_OK;
}

}  // extern "C"
