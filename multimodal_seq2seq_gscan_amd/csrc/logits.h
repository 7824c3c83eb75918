// Rows of logits: what the kernels over a vocabulary share (top_logits.hip, distill.hip, beam.hip).
//
// A row is V words of float, bfloat16 or half, its words adjacent; rows lie [outer][inner] with a stride each, in elements
// (gscan_rows), so that a slice of a longer batch is read in place.  A row may begin at any element: 16-byte loads and
// stores need no more than the element's own alignment in global memory on gfx950, so there is one path for every
// alignment instead of a scalar head per row.
#pragma once
#include <float.h>
#include <string.h>

#include "common.h"
#include "gscan_hip.h"

namespace gscan {

// ---- host side: argument checks and entry points (capi.hip calls these) ----
int check_rows(const char *who, const gscan_rows *rows);
size_t top_logits_workspace(const gscan_rows &rows, int K);
int top_logits(const gscan_rows &rows, int K, void *values, int32_t *indices, float *lse, void *workspace, size_t bytes,
               hipStream_t stream);
size_t distillation_workspace(const gscan_rows &rows);
int distillation_loss(const gscan_rows &rows, const gscan_distillation &terms, const float *upstream, void *grad, float *loss,
                      float *stats, void *workspace, size_t bytes, hipStream_t stream);
size_t beam_select_workspace(const gscan_rows &rows);
int beam_select(const gscan_rows &rows, const float *scores, const uint8_t *finished, int eos, int pad, float *scores_out,
                int32_t *parents, int64_t *tokens, uint8_t *finished_out, void *workspace, size_t bytes, hipStream_t stream);
int beam_reorder(int B, int W, const int32_t *parents, const gscan_state *states, int count, hipStream_t stream);

constexpr int kMaxTop = 256;       // entries a row's selection or a teacher's row may hold
constexpr int kMaxBeams = 64;
constexpr float kLog2e = 1.4426950408889634f;

// A selection of the top K of every row (or of every chunk of a row), and what the beam step takes from it.
struct TopChunks { int splits, chunk; };
TopChunks top_chunks(const gscan_rows &rows, int K);
// part of a row's softmax sum: sum = sum exp(z - ref) over the chunk, in 64 bits (candidates of different beams are compared
// through it)
struct LsePart { double sum; float ref; float unused; };
// keys [row][split][K] (sorted, 0 = no entry) and lse parts [row][split]; rows with skip[row] set are left out
int top_chunk_keys(const gscan_rows &rows, int K, TopChunks c, uint64_t *keys, LsePart *lse, const uint8_t *finished,
                   const float *scores, hipStream_t stream);

#if defined(__HIPCC__)
struct TypeF32 { static constexpr int bytes = 4, vec = 4; };
struct TypeBF16 { static constexpr int bytes = 2, vec = 8; };
struct TypeF16 { static constexpr int bytes = 2, vec = 8; };

struct Rows {                     // gscan_rows as the kernels take it
    const char *data;
    int64_t so, si;               // bytes
    int inner, V;
    __device__ __forceinline__ const char *row(int r) const {
        const int o = r / inner;
        return data + (int64_t)o * so + (int64_t)(r - o * inner) * si;
    }
};
static inline Rows device_rows(const gscan_rows &r) {
    const int b = r.type == GSCAN_F32 ? 4 : 2;
    return Rows{(const char *)r.data, r.stride_outer * b, r.stride_inner * b, (int)r.inner, r.V};
}

struct Raw { uint32_t w[4]; };    // 16 bytes of a row

typedef uint32_t Quad2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t Quad4 __attribute__((ext_vector_type(4), aligned(4)));

template <class T, bool STREAM = false>
__device__ __forceinline__ Raw load16(const char *p) {
    Quad2 q;
    if constexpr (STREAM) {
        if constexpr (T::bytes == 4) q = __builtin_nontemporal_load((const Quad4 *)p);
        else q = __builtin_nontemporal_load((const Quad2 *)p);
    } else {
        if constexpr (T::bytes == 4) q = *(const Quad4 *)p;
        else q = *(const Quad2 *)p;
    }
    return Raw{{q.x, q.y, q.z, q.w}};
}
template <class T, bool STREAM = false>
__device__ __forceinline__ void store16(char *p, const Raw &r) {
    const Quad2 q = {r.w[0], r.w[1], r.w[2], r.w[3]};
    if constexpr (T::bytes == 4) {
        if constexpr (STREAM) __builtin_nontemporal_store((Quad4)q, (Quad4 *)p);
        else *(Quad4 *)p = q;
    } else {
        if constexpr (STREAM) __builtin_nontemporal_store(q, (Quad2 *)p);
        else *(Quad2 *)p = q;
    }
}

__device__ __forceinline__ float half_bits(uint32_t b) { _Float16 h; const uint16_t s = (uint16_t)b; __builtin_memcpy(&h, &s, 2); return (float)h; }
__device__ __forceinline__ uint32_t to_half_bits(float f) { const _Float16 h = (_Float16)f; uint16_t s; __builtin_memcpy(&s, &h, 2); return s; }
// round to nearest even; a NaN stays one
__device__ __forceinline__ uint32_t to_bf16_bits(float f) {
    const __bf16 h = (__bf16)f;
    uint16_t s;
    __builtin_memcpy(&s, &h, 2);
    return s;
}

// element e (a compile-time number) of 16 loaded bytes
template <class T>
__device__ __forceinline__ float element(const Raw &r, int e) {
    if constexpr (T::bytes == 4) return __uint_as_float(r.w[e]);
    const uint32_t w = r.w[e >> 1];
    if constexpr (__is_same(T, TypeBF16)) return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
    return half_bits((e & 1) ? (w >> 16) : (w & 0xffffu));
}
template <class T>
__device__ __forceinline__ Raw pack(const float (&x)[T::vec]) {
    Raw r;
    if constexpr (T::bytes == 4) {
        for (int i = 0; i < 4; ++i) r.w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (__is_same(T, TypeBF16)) r.w[i] = to_bf16_bits(x[2 * i]) | (to_bf16_bits(x[2 * i + 1]) << 16);
            else r.w[i] = to_half_bits(x[2 * i]) | (to_half_bits(x[2 * i + 1]) << 16);
        }
    }
    return r;
}
// one element of a row
template <class T>
__device__ __forceinline__ float load1(const char *row, int i) {
    if constexpr (T::bytes == 4) return *(const float *)(row + (int64_t)i * 4);
    const uint32_t b = *(const uint16_t *)(row + (int64_t)i * 2);
    if constexpr (__is_same(T, TypeBF16)) return __uint_as_float(b << 16);
    return half_bits(b);
}
template <class T>
__device__ __forceinline__ void store1(char *row, int64_t i, float f) {
    if constexpr (T::bytes == 4) *(float *)(row + i * 4) = f;
    else if constexpr (__is_same(T, TypeBF16)) *(uint16_t *)(row + i * 2) = (uint16_t)to_bf16_bits(f);
    else *(uint16_t *)(row + i * 2) = (uint16_t)to_half_bits(f);
}
// a partial group of words at a row's end: words behind the row read as -inf
template <class T>
__device__ __forceinline__ Raw load_tail(const char *row, int first, int n) {
    Raw r;
    if constexpr (T::bytes == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = first + i < n ? *(const uint32_t *)(row + (int64_t)(first + i) * 4) : 0xff800000u;
    } else {
        constexpr uint32_t ninf = __is_same(T, TypeBF16) ? 0xff80u : 0xfc00u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = first + 2 * i;
            const uint32_t lo = j < n ? *(const uint16_t *)(row + (int64_t)j * 2) : ninf;
            const uint32_t hi = j + 1 < n ? *(const uint16_t *)(row + (int64_t)(j + 1) * 2) : ninf;
            r.w[i] = lo | (hi << 16);
        }
    }
    return r;
}
template <class T>
__device__ __forceinline__ Raw load_group(const char *row, int g, int n) {     // words [g vec, g vec + vec) of n
    const int first = g * T::vec;
    return first + T::vec <= n ? load16<T>(row + (int64_t)first * T::bytes) : load_tail<T>(row, first, n);
}

// Whole numbers that order floats by value; a NaN counts as -inf, -0 as +0.  0 stands for "no element" (-inf has 0x007fffff).
__device__ __forceinline__ uint32_t order_key(float f) {
    f = fmaxf(f, -INFINITY) + 0.0f;
    const uint32_t u = __float_as_uint(f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t order_key64(double d) {
    const uint64_t u = (uint64_t)__double_as_longlong(d + 0.0);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
// (value, index) as one number: larger = earlier in the order (value descending, index ascending); 0 = no entry.  62 bits, an
// index being below 2^30: also as a double's bits the numbers are in order (positive, finite), and two doubles are compared at
// several times the rate of two 64-bit integers.
__device__ __forceinline__ uint64_t pair_key(uint32_t key, int index) { return ((uint64_t)key << 30) | (0x3fffffffu - (uint32_t)index); }
__device__ __forceinline__ uint32_t pair_value(uint64_t x) { return (uint32_t)(x >> 30); }
__device__ __forceinline__ int pair_index(uint64_t x) { return (int)(0x3fffffffu - ((uint32_t)x & 0x3fffffffu)); }
__device__ __forceinline__ double pair_double(uint64_t x) { return __longlong_as_double((int64_t)x); }

template <typename V, class Op>
__device__ __forceinline__ V wave_reduce(V v, Op op) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = op(v, __shfl_xor(v, d));
    return v;
}

// The same over groups of L = 4, 8 or 16 lanes, on the DPP datapath.  All lanes must be active.
template <int CTRL, typename V>
__device__ __forceinline__ V dpp_word(V v) {
    static_assert(sizeof(V) == 4 || sizeof(V) == 8, "one word or two");
    int w[sizeof(V) / 4];
    __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
    for (int i = 0; i < (int)sizeof(V) / 4; ++i) w[i] = __builtin_amdgcn_update_dpp(0, w[i], CTRL, 0xf, 0xf, false);
    __builtin_memcpy(&v, w, sizeof(V));
    return v;
}
template <int L, typename V, class Op>
__device__ __forceinline__ V group_reduce(V v, Op op) {
    v = op(v, dpp_word<0xb1>(v));                          // quad_perm [1,0,3,2]
    v = op(v, dpp_word<0x4e>(v));                          // quad_perm [2,3,0,1]
    if constexpr (L > 4) v = op(v, dpp_word<0x141>(v));    // row_half_mirror
    if constexpr (L > 8) v = op(v, dpp_word<0x140>(v));    // row_mirror
    return v;
}
// how many of the sixteen lanes' numbers come before this lane's
__device__ __forceinline__ int sum_before16(int v) {
    int s = v;
    s += dpp_word<0x111>(s);                               // row_shr:1, 2, 4, 8: 0 from outside the row
    s += dpp_word<0x112>(s);
    s += dpp_word<0x114>(s);
    s += dpp_word<0x118>(s);
    return s - v;
}

// log sum exp from the parts of a row's chunks, in 64 bits; one wave.
__device__ __forceinline__ double join_lse(const LsePart *part, int n) {
    const int lane = threadIdx.x & 63;
    float ref = -FLT_MAX;
    for (int i = lane; i < n; i += 64) ref = fmaxf(ref, part[i].ref);
    ref = wave_reduce(ref, [](float a, float b) { return fmaxf(a, b); });
    double s = 0.0;
    for (int i = lane; i < n; i += 64) s += part[i].sum * exp((double)part[i].ref - (double)ref);
    s = wave_reduce(s, [](double a, double b) { return a + b; });
    return ref == INFINITY ? (double)INFINITY : (double)ref + log(s);
}

// A number t such that at least K of n keys in LDS are >= t, and (unless many are equal) few more than K: bisection between
// the keys' least and largest, counting with ballots; it ends as soon as the count is within K .. K + K/4, or the interval is
// one number.  One wave, n <= 64 * SLOTS.  With fewer than K keys > 0 the answer is 0.
// `keys(i)` reads the i-th.
template <int SLOTS, class F>
__device__ __forceinline__ uint32_t kth_bound(F keys, int n, int K, int lane) {
    uint32_t k[SLOTS], hi = 0, lo = ~0u;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        k[i] = lane + 64 * i < n ? keys(lane + 64 * i) : 0u;
        hi = max(hi, k[i]);
        if (k[i]) lo = min(lo, k[i]);
    }
    auto count = [&](uint32_t least) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) c += __popcll(__ballot(k[i] >= least));
        return c;
    };
    if (count(1) < K) return 0;
    // count(>= lo) >= K and count(>= top) < K throughout; a lane's largest key bounds from below too where K <= 64 lanes
    const uint32_t least = K <= 64 && __ballot(hi != 0) == ~0ull ? hi : lo;
    lo = __builtin_amdgcn_readfirstlane(wave_reduce(least, [](uint32_t a, uint32_t b) { return min(a, b); }));
    hi = __builtin_amdgcn_readfirstlane(wave_reduce(hi, [](uint32_t a, uint32_t b) { return max(a, b); }));
    const int most = K + (K >> 2);
    uint32_t top = hi + 1;       // keys of numbers end far below 2^32 - 1
    while (top - lo > 1) {
        const uint32_t mid = lo + (top - lo) / 2;
        const int c = count(mid);
        if (c >= K) {
            lo = mid;
            if (c <= most) break;
        } else {
            top = mid;
        }
    }
    return lo;
}
#endif

}  // namespace gscan
