// Distillation from a teacher's top logits (and the hard loss beside it) over rows of logits, with the gradient.
//
//   p = softmax over a row's K teacher entries of t / tau,  q = softmax(z / tau),  s = softmax(z),  over the live rows:
//   loss  = scale * sum_rows [ hard (lse z - z_y) + soft tau^2 sum_k p_k (log p_k - log q[idx_k]) ]
//   d/dz_v = scale * [ hard (s_v - [v = y]) + soft tau (q_v - sum_{k: idx_k = v} p_k) ],   scale = 1 / live rows, or 1
//
// A row is read once: it stays in registers, as it came (16-byte pieces), between the two reductions (its maximum, its sums)
// and the gradient.  The exponentials are taken a second time for the gradient: holding them would take twice the registers
// for 16-bit words.  sum_k p_k (log p_k - log q_k) needs no normalisers inside: with e_k = exp((t_k - t_max) / tau) and
// A = sum e, B = sum e_k ((t_k - t_max) - (z_k - z_max)) / tau it is B / A - log A + log sum exp((z - z_max) / tau), so
// one more reduction beside the row's sums does it.  Sums are in 32 bits within a row and in 64 across rows.
// The few words that the teacher or the label names are stored a second time behind the row, with their share taken off:
// same workgroup, behind a barrier; an index that comes twice is handled once, by its first entry, with both shares.
#include "logits.h"

namespace gscan {

namespace {
constexpr int kCountBlocks = 64;

struct DistillArgs {
    Rows rows;
    int count;                         // rows in all
    const void *indices; int index_bits;
    const void *teacher; int teacher_type;
    int K;
    const int64_t *labels; int64_t ignore; int shift;
    float inv_tau, soft, hard;
    float soft_grad;                   // soft weight times tau
    const int *live;                   // kCountBlocks partial counts (mean), or NULL (sum)
    const float *upstream;             // or NULL: 1
    char *grad;                        // [rows][V], or NULL
    double *part;                      // [workgroups][3]: hard loss, soft loss, live rows
};

// the label of row r, or -1 when the row is not live; -2 when there are no labels and every row is
__device__ __forceinline__ int row_label(const DistillArgs &a, int r) {
    if (!a.labels) return -2;
    int64_t y;
    if (a.shift) y = (r + 1) % a.rows.inner ? a.labels[r + 1] : (int64_t)0;       // the sequence moved left by one, 0 behind it
    else y = a.labels[r];
    return y != a.ignore && y >= 0 && y < a.rows.V ? (int)y : -1;
}

__device__ __forceinline__ float teacher_value(const DistillArgs &a, int64_t at) {
    if (a.teacher_type == GSCAN_F32) return load1<TypeF32>((const char *)a.teacher + at * 4, 0);
    const char *p = (const char *)a.teacher + at * 2;
    return a.teacher_type == GSCAN_BF16 ? load1<TypeBF16>(p, 0) : load1<TypeF16>(p, 0);
}
// an index outside [0, V) is no entry: -1
__device__ __forceinline__ int teacher_index(const DistillArgs &a, int64_t at) {
    const int64_t i = a.index_bits == 64 ? ((const int64_t *)a.indices)[at] : (int64_t)((const int32_t *)a.indices)[at];
    return i >= 0 && i < a.rows.V ? (int)i : -1;
}

// 1 / live rows (or 1) times the upstream gradient; every lane of the wave takes part
__device__ __forceinline__ float gradient_scale(const DistillArgs &a) {
    float s = a.upstream ? a.upstream[0] : 1.f;
    if (a.live) {
        const int n = wave_reduce(a.live[threadIdx.x & 63], [](int x, int y) { return x + y; });
        s = n > 0 ? s / (float)n : 0.f;
    }
    return s;
}

// live rows, in kCountBlocks parts
__global__ __launch_bounds__(256) void distill_count_kernel(DistillArgs a, int *live) {
    __shared__ int s[4];
    int n = 0;
    for (int r = blockIdx.x * 256 + threadIdx.x; r < a.count; r += kCountBlocks * 256) n += row_label(a, r) != -1 ? 1 : 0;
    n = wave_reduce(n, [](int x, int y) { return x + y; });
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) live[blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}

// stats: hard loss sum, live rows, soft loss sum (with tau^2), loss
__global__ __launch_bounds__(1024) void distill_finish_kernel(const double *part, int n, float soft, float hard, int mean, float *stats) {
    __shared__ double s[3][16];
    double v[3] = {0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < n; i += 1024) {
        v[0] += part[3 * (int64_t)i]; v[1] += part[3 * (int64_t)i + 1]; v[2] += part[3 * (int64_t)i + 2];
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        v[k] = wave_reduce(v[k], [](double x, double y) { return x + y; });
        if ((threadIdx.x & 63) == 0) s[k][threadIdx.x >> 6] = v[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 0; k < 3; ++k) {
            v[k] = s[k][0];
            for (int w = 1; w < 16; ++w) v[k] += s[k][w];
        }
        const double loss = (hard != 0.f ? (double)hard * v[0] : 0.0) + (soft != 0.f ? (double)soft * v[1] : 0.0);
        stats[0] = (float)v[0]; stats[1] = (float)v[2]; stats[2] = (float)v[1];
        stats[3] = (float)(mean ? loss / (v[2] > 0.0 ? v[2] : 1.0) : loss);
    }
}

template <int TPB>
struct RowShared {
    int index[kMaxTop + 1];
    float share[kMaxTop + 1];        // e_k
    float red[5][TPB / 64 + 1];
};

template <int TPB, int N, class Op>
__device__ __forceinline__ void block_reduce(RowShared<TPB> &sh, float (&v)[N], Op op) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_reduce(v[i], op);
    if constexpr (TPB > 64) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) sh.red[i][wave] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = sh.red[i][0];
            for (int w = 1; w < TPB / 64; ++w) v[i] = op(v[i], sh.red[i][w]);
        }
        __syncthreads();
    }
}

// One workgroup per row.  NR > 0: the row in NR 16-byte pieces per thread; NR = 0: the row is read again for every use (rows
// longer than the registers of a workgroup of 1024).
// TWO: two different exponentials a word (both terms, tau != 1); otherwise one serves the term or both.
template <class T, int TPB, int NR, bool TWO, bool GRAD>
__global__ __launch_bounds__(TPB) void distill_row_kernel(DistillArgs a) {
    __shared__ RowShared<TPB> sh;
    constexpr int NK = TPB >= kMaxTop ? 1 : kMaxTop / TPB;      // teacher entries per thread
    const int tid = threadIdx.x, r = blockIdx.x, V = a.rows.V;
    const char *row = a.rows.row(r);
    const int pieces = V / T::vec, rest = V - pieces * T::vec;       // whole 16-byte pieces, and words behind them: one a thread
    const int label = row_label(a, r);
    char *out = GRAD ? a.grad + (int64_t)r * V * T::bytes : nullptr;
    if (label == -1) {                 // not live: neither its words nor its teacher's are read
        if constexpr (GRAD) {
            for (int p = tid; p < pieces; p += TPB) store16<T>(out + (int64_t)p * 16, Raw{{0, 0, 0, 0}});
            if (tid < rest) store1<T>(out, pieces * T::vec + tid, 0.f);
        }
        if (tid == 0) { a.part[3 * (int64_t)r] = 0.0; a.part[3 * (int64_t)r + 1] = 0.0; a.part[3 * (int64_t)r + 2] = 0.0; }
        return;
    }
    Raw x[NR ? NR : 1];
#pragma unroll
    for (int i = 0; i < NR; ++i)
        if (i * TPB < pieces) x[i] = load16<T>(row + (int64_t)min(tid + i * TPB, pieces - 1) * 16);
    const float last = tid < rest ? load1<T>(row, pieces * T::vec + tid) : -INFINITY;
    // f(16 bytes, piece number) for every piece of this thread
    auto each = [&](auto f) {
        if constexpr (NR > 0) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
                if (i * TPB < pieces && tid + i * TPB < pieces) f(x[i], tid + i * TPB);
        } else {
            for (int p = tid; p < pieces; p += TPB) f(load16<T>(row + (int64_t)p * 16), p);
        }
    };

    // The compiler would keep the widened words from one use to the next (twice the registers for 16-bit words, and spills):
    // behind this the pieces are new values to it.
    auto hide = [&]() {
#pragma unroll
        for (int i = 0; i < NR; ++i) asm volatile("" : "+v"(x[i].w[0]), "+v"(x[i].w[1]), "+v"(x[i].w[2]), "+v"(x[i].w[3]));
    };

    int idx[NK];
    float t[NK], zk[NK];
    float top[2] = {-INFINITY, -INFINITY};        // of the row, of the teacher's entries
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        const int k = tid + j * TPB;
        idx[j] = -1; t[j] = -INFINITY; zk[j] = 0.f;
        if (k < a.K) {
            const int64_t at = (int64_t)r * a.K + k;
            idx[j] = teacher_index(a, at);
            if (idx[j] >= 0) { t[j] = teacher_value(a, at); zk[j] = load1<T>(row, idx[j]); }
            sh.index[k] = idx[j];
        }
        top[1] = fmaxf(top[1], t[j]);
    }
    const float zy = label >= 0 ? load1<T>(row, label) : 0.f;
    each([&](const Raw &w, int) {
#pragma unroll
        for (int e = 0; e < T::vec; ++e) top[0] = fmaxf(top[0], element<T>(w, e));
    });
    top[0] = fmaxf(top[0], last);
    block_reduce<TPB>(sh, top, [](float p, float q) { return fmaxf(p, q); });
    hide();
    const float zmax = top[0], tmax = top[1];

    // exponents in powers of two, of the distance from the maximum: finite also where every word is the type's lowest
    const float a0 = (TWO || a.soft != 0.f ? a.inv_tau : 1.f) * kLog2e, a1 = kLog2e;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};         // sum of the first exponential, of the second, A, B
    each([&](const Raw &w, int) {
#pragma unroll
        for (int e = 0; e < T::vec; ++e) {
            const float d = element<T>(w, e) - zmax;
            sums[0] += __builtin_amdgcn_exp2f(d * a0);
            if constexpr (TWO) sums[1] += __builtin_amdgcn_exp2f(d * a1);
        }
    });
    if (tid < rest) {
        sums[0] += __builtin_amdgcn_exp2f((last - zmax) * a0);
        if constexpr (TWO) sums[1] += __builtin_amdgcn_exp2f((last - zmax) * a1);
    }
    float share[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        const int k = tid + j * TPB;
        const float d = (t[j] - tmax) * a.inv_tau;
        share[j] = idx[j] >= 0 && t[j] != -INFINITY ? __builtin_amdgcn_exp2f(d * kLog2e) : 0.f;
        if (share[j] != 0.f) {
            sums[2] += share[j];
            sums[3] += share[j] * (d - (zk[j] - zmax) * a.inv_tau);
        }
        if (k < a.K) sh.share[k] = share[j];
    }
    block_reduce<TPB>(sh, sums, [](float p, float q) { return p + q; });
    const float s0 = sums[0], s1 = TWO ? sums[1] : sums[0], A = sums[2], B = sums[3];
    if (tid == 0) {
        const float hard = a.hard != 0.f ? logf(s1) - (zy - zmax) : 0.f;
        const float soft = a.soft != 0.f && A != 0.f ? B / A - logf(A) + logf(s0) : 0.f;
        a.part[3 * (int64_t)r] = (double)hard;
        a.part[3 * (int64_t)r + 1] = (double)soft;
        a.part[3 * (int64_t)r + 2] = 1.0;
    }
    if constexpr (GRAD) {
        hide();
        const float scale = gradient_scale(a);
        const float soft = a.soft != 0.f && A != 0.f ? a.soft_grad * scale : 0.f, hard = a.hard != 0.f ? a.hard * scale : 0.f;
        const float c0 = TWO ? soft / s0 : (soft + hard) / s0, c1 = TWO ? hard / s1 : 0.f;
        auto density = [&](float z) {
            const float d = z - zmax;
            float g = c0 * __builtin_amdgcn_exp2f(d * a0);
            if constexpr (TWO) g = fmaf(c1, __builtin_amdgcn_exp2f(d * a1), g);
            return g;
        };
        each([&](const Raw &w, int p) {
            float g[T::vec];
#pragma unroll
            for (int e = 0; e < T::vec; ++e) g[e] = density(element<T>(w, e));
            store16<T>(out + (int64_t)p * 16, pack<T>(g));
        });
        if (tid < rest) store1<T>(out, pieces * T::vec + tid, density(last));
        __syncthreads();                 // the row is stored: the named words follow
        const float soft_share = A != 0.f ? soft / A : 0.f;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const int k = tid + j * TPB;
            if (k >= a.K || idx[j] < 0) continue;
            float named = 0.f;
            bool first = true;
            for (int i = 0; i < a.K; ++i)
                if (sh.index[i] == idx[j]) { first = first && i >= k; named += sh.share[i]; }
            if (first) store1<T>(out, idx[j], density(zk[j]) - soft_share * named - (idx[j] == label ? hard : 0.f));
        }
        if (tid == 0 && label >= 0 && hard != 0.f) {
            bool named = false;
            for (int i = 0; i < a.K; ++i) named = named || sh.index[i] == label;
            if (!named) store1<T>(out, label, density(zy) - hard);
        }
    }
}

// Vocabularies of at most 64 words: L lanes per row, a word per lane; the teacher's entries of a workgroup's rows in LDS.
template <class T, int L, bool GRAD>
__global__ __launch_bounds__(256) void distill_small_kernel(DistillArgs a) {
    extern __shared__ float entries[];
    __shared__ double s_part[4][3];
    constexpr int R = 256 / L;
    const int slot = threadIdx.x / L, v = threadIdx.x & (L - 1), r = blockIdx.x * R + slot, V = a.rows.V, K = a.K;
    float *share = entries + slot * K;
    int8_t *index = (int8_t *)(entries + R * K) + slot * K;      // at most 64 words
    const int label = r < a.count ? row_label(a, r) : -1;
    const bool live = label != -1, in = live && v < V;
    const char *row = a.rows.row(r < a.count ? r : 0);
    const float z = in ? load1<T>(row, v) : -INFINITY;
    auto lanes = [](float x, auto op) {
#pragma unroll
        for (int d = L / 2; d; d >>= 1) x = op(x, __shfl_xor(x, d, L));
        return x;
    };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto plus = [](float x, float y) { return x + y; };
    const float zmax = lanes(z, larger);
    float tmax = -INFINITY;
    for (int k = v; k < K; k += L) {
        const int64_t at = (int64_t)r * K + k;
        const int i = live ? teacher_index(a, at) : -1;
        const float t = i >= 0 ? teacher_value(a, at) : -INFINITY;
        index[k] = (int8_t)i; share[k] = t;
        tmax = fmaxf(tmax, t);
    }
    tmax = lanes(tmax, larger);
    const bool soft_on = a.soft != 0.f, hard_on = a.hard != 0.f;
    float A = 0.f, B = 0.f;
    for (int k = v; k < K; k += L) {
        const float t = share[k], d = (t - tmax) * a.inv_tau;
        const int i = index[k];
        float e = 0.f;
        if (i >= 0 && t != -INFINITY) {
            e = __builtin_amdgcn_exp2f(d * kLog2e);
            if (e != 0.f) { A += e; B += e * (d - (load1<T>(row, i) - zmax) * a.inv_tau); }
        }
        share[k] = e;
    }
    A = lanes(A, plus);
    B = lanes(B, plus);
    const float e0 = in ? __builtin_amdgcn_exp2f((z - zmax) * a.inv_tau * kLog2e) : 0.f;
    const float e1 = in ? __builtin_amdgcn_exp2f((z - zmax) * kLog2e) : 0.f;
    const float s0 = lanes(e0, plus), s1 = lanes(e1, plus);
    const float zy = label >= 0 ? __shfl(z, label, L) : 0.f;
    if constexpr (GRAD) {
        const float scale = gradient_scale(a);
        float g = 0.f;
        if (in) {
            if (hard_on) g = a.hard * scale * (e1 / s1 - (v == label ? 1.f : 0.f));
            if (soft_on && A != 0.f) {
                float named = 0.f;
                for (int k = 0; k < K; ++k) named += index[k] == v ? share[k] : 0.f;
                g += a.soft_grad * scale * (e0 / s0 - named / A);
            }
        }
        if (r < a.count && v < V) store1<T>(a.grad, (int64_t)r * V + v, g);
    }
    double part[3] = {0.0, 0.0, 0.0};
    if (live && v == 0) {
        part[0] = hard_on ? (double)(logf(s1) - (zy - zmax)) : 0.0;
        part[1] = soft_on && A != 0.f ? (double)(B / A - logf(A) + logf(s0)) : 0.0;
        part[2] = 1.0;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        part[k] = wave_reduce(part[k], [](double x, double y) { return x + y; });
        if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6][k] = part[k];
    }
    __syncthreads();
    if (threadIdx.x < 3)
        a.part[3 * (int64_t)blockIdx.x + threadIdx.x] =
            s_part[0][threadIdx.x] + s_part[1][threadIdx.x] + s_part[2][threadIdx.x] + s_part[3][threadIdx.x];
}

int small_lanes(int V) { return V <= 8 ? 8 : V <= 16 ? 16 : V <= 32 ? 32 : 64; }
int part_blocks(const gscan_rows &rows) {
    const int64_t n = rows.outer * rows.inner;
    return rows.V <= 64 ? cdiv(n, 256 / small_lanes(rows.V)) : (int)n;
}

template <class T, int L>
int launch_small(const DistillArgs &a, hipStream_t stream) {
    const int blocks = cdiv(a.count, 256 / L);
    const size_t lds = (size_t)(256 / L) * a.K * 5;
    if (a.grad) hipLaunchKernelGGL((distill_small_kernel<T, L, true>), dim3(blocks), dim3(256), lds, stream, a);
    else hipLaunchKernelGGL((distill_small_kernel<T, L, false>), dim3(blocks), dim3(256), lds, stream, a);
    GSCAN_LAUNCHED("distill_small_kernel");
    return 0;
}

template <class T, int TPB, int NR>
int launch_row(const DistillArgs &a, bool two, hipStream_t stream) {
    const dim3 grid(a.count), block(TPB);
    if (two && a.grad) hipLaunchKernelGGL((distill_row_kernel<T, TPB, NR, true, true>), grid, block, 0, stream, a);
    else if (two) hipLaunchKernelGGL((distill_row_kernel<T, TPB, NR, true, false>), grid, block, 0, stream, a);
    else if (a.grad) hipLaunchKernelGGL((distill_row_kernel<T, TPB, NR, false, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((distill_row_kernel<T, TPB, NR, false, false>), grid, block, 0, stream, a);
    GSCAN_LAUNCHED("distill_row_kernel");
    return 0;
}

template <class T>
int launch_type(const DistillArgs &a, hipStream_t stream) {
    const int V = a.rows.V;
    if (V <= 64) {
        switch (small_lanes(V)) {
            case 8: return launch_small<T, 8>(a, stream);
            case 16: return launch_small<T, 16>(a, stream);
            case 32: return launch_small<T, 32>(a, stream);
            default: return launch_small<T, 64>(a, stream);
        }
    }
    const bool two = a.hard != 0.f && a.soft != 0.f && a.inv_tau != 1.f;
    const int pieces = V / T::vec;
    if (pieces <= 64 * 8) return launch_row<T, 64, 8>(a, two, stream);
    if (pieces <= 256 * 16) return launch_row<T, 256, 16>(a, two, stream);
    if (pieces <= 512 * 16) return launch_row<T, 512, 16>(a, two, stream);
    if (pieces <= 1024 * 16) return launch_row<T, 1024, 16>(a, two, stream);
    return launch_row<T, 1024, 0>(a, two, stream);
}
}  // namespace

size_t distillation_workspace(const gscan_rows &rows) {
    return kCountBlocks * sizeof(int) + (size_t)part_blocks(rows) * 3 * sizeof(double);
}

int distillation_loss(const gscan_rows &rows, const gscan_distillation &t, const float *upstream, void *grad, float *stats,
                      void *workspace, size_t bytes, hipStream_t stream) {
    GSCAN_CHECK(stats, "distillation_loss: stats is NULL");
    GSCAN_CHECK(t.K >= 1 && t.K <= kMaxTop, "distillation_loss: %d teacher entries per row (1 to %d)", t.K, kMaxTop);
    GSCAN_CHECK(t.indices && t.teacher, "distillation_loss: the teacher's indices or logits are NULL");
    GSCAN_CHECK(t.index_bits == 32 || t.index_bits == 64, "distillation_loss: %d bits per index (32 or 64)", t.index_bits);
    GSCAN_CHECK(t.teacher_type == GSCAN_F32 || t.teacher_type == GSCAN_BF16 || t.teacher_type == GSCAN_F16,
                "distillation_loss: unknown type %d of the teacher's logits", t.teacher_type);
    GSCAN_CHECK(t.temperature >= 1e-3f && t.temperature <= 1e3f, "distillation_loss: temperature %g (1e-3 to 1e3)", (double)t.temperature);
    GSCAN_CHECK(t.soft_weight >= 0.f && t.soft_weight <= FLT_MAX && t.hard_weight >= 0.f && t.hard_weight <= FLT_MAX,
                "distillation_loss: weights %g (soft) and %g (hard): finite and not negative", (double)t.soft_weight, (double)t.hard_weight);
    GSCAN_CHECK(t.labels || t.hard_weight == 0.f, "distillation_loss: a hard loss needs labels");
    const size_t need = distillation_workspace(rows);
    GSCAN_CHECK(workspace && bytes >= need, "distillation_loss: workspace of %zu bytes, %zu needed", workspace ? bytes : (size_t)0, need);
    GSCAN_CHECK((uintptr_t)workspace % 8 == 0, "distillation_loss: workspace is not aligned to 8 bytes");
    const int b = rows.type == GSCAN_F32 ? 4 : 2;
    GSCAN_CHECK((uintptr_t)grad % b == 0, "distillation_loss: the gradient is not aligned to its type");
    int *live = (int *)workspace;
    DistillArgs a{};
    a.rows = device_rows(rows);
    a.count = (int)(rows.outer * rows.inner);
    a.indices = t.indices; a.index_bits = t.index_bits; a.teacher = t.teacher; a.teacher_type = t.teacher_type; a.K = t.K;
    a.labels = t.labels; a.ignore = t.ignore_index; a.shift = t.shift_labels != 0;
    a.inv_tau = 1.f / t.temperature;
    a.soft = t.soft_weight; a.soft_grad = t.soft_weight * t.temperature; a.hard = t.hard_weight;
    a.upstream = upstream; a.grad = (char *)grad;
    a.part = (double *)(live + kCountBlocks);
    if (grad && !t.sum_reduction) {       // the gradient of a mean needs the number of live rows first
        a.live = live;
        hipLaunchKernelGGL(distill_count_kernel, dim3(kCountBlocks), dim3(256), 0, stream, a, live);
        GSCAN_LAUNCHED("distill_count_kernel");
    }
    const int type = rows.type;
    TRY_RC(type == GSCAN_F32 ? launch_type<TypeF32>(a, stream) : type == GSCAN_BF16 ? launch_type<TypeBF16>(a, stream)
                                                                                   : launch_type<TypeF16>(a, stream));
    const float tau2 = t.temperature * t.temperature;
    hipLaunchKernelGGL(distill_finish_kernel, dim3(1), dim3(1024), 0, stream, a.part, part_blocks(rows), t.soft_weight * tau2,
                       t.hard_weight, t.sum_reduction ? 0 : 1, stats);
    GSCAN_LAUNCHED("distill_finish_kernel");
    return 0;
}

}  // namespace gscan
