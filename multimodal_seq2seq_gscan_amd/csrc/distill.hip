// Distillation from a teacher's top logits (and the hard loss beside it) over rows of logits, with the gradient.
//
//   p = softmax over a row's K teacher entries of t / tau,  q = softmax(z / tau),  s = softmax(z),  over the live rows:
//   loss  = scale * sum_rows [ hard (lse z - z_y) + soft tau^2 sum_k p_k (log p_k - log q[idx_k]) ]
//   d/dz_v = scale * [ hard (s_v - [v = y]) + soft tau (q_v - sum_{k: idx_k = v} p_k) ],   scale = 1 / live rows, or 1
//
// A row is read once: it stays in registers, as it came (16-byte pieces), between the two reductions (its maximum, its sums)
// and the gradient.  The exponentials are taken a second time for the gradient: holding them would take twice the registers
// for 16-bit words.  sum_k p_k (log p_k - log q_k) needs no normalisers inside: with e_k = exp((t_k - t_max) / tau) and
// A = sum e, B = sum e_k ((t_k - t_max) - (z_k - z_max)) it is B / (A tau) + log(sum exp((z - z_max) / tau) / A), so
// one more reduction beside the row's sums does it; the same rounded 1 / tau stands in p, q and B: it changes the temperature,
// not the difference.  Sums are in 32 bits within a row and in 64 across rows.
// The few words that the teacher or the label names are stored a second time behind the row, with their share taken off:
// same workgroup, behind a barrier; an index that comes twice is handled once, by its first entry, with both shares.
#include <type_traits>

#include "logits.h"

namespace gscan {

namespace {
constexpr int kCountBlocks = 64;
// Up to so many rows, the launch that needs the number of live rows counts the labels itself, in every workgroup; above, a launch
// before it does.  Short rows (9 words of float), counted inside / before, kernels back to back and whole calls, which the host
// binds: 1024 rows 9.4 / 10.8 and 21.5 / 23.8 us, 4096: 10.9 / 10.9 and 21.3 / 23.6, 8192: 12.9 / 11.0 and 21.3 / 23.8, 16384: 17.2 /
// 11.1 and 21.3 / 23.6, 32768: 25.5 / 11.7 and 25.7 / 23.7: between 4096 and 16384 rows the launch before is better in a replayed
// graph's chain of kernels, the count inside from the host, which launches a kernel less.  Long rows, which fill the chip with workgroups: 2000 words, 256 rows 10.9 / 12.5 us, 1024:
// 14.9 / 14.8, 2048: 20.8 / 19.2; 32000 words, 256 rows 24.0 / 25.7, 1024: 57.9 / 58.8.
constexpr int kCountThere = 8192, kCountThereLong = 256;
// Above so many workgroups their parts are added up by 64 workgroups before the one that finishes.  Without / with that launch,
// kernels back to back: 8192 parts 54.3 / 54.4 us (131072 rows of 100 words, 16 rows a workgroup) and 32.4 / 32.6 (rows of 1030
// words), 16384: 95.7 / 93.6 and 49.2 / 47.0, 32768: 184.0 / 177.2 and 83.7 / 77.2; 4096: 34.0 / 35.3 and 21.0 / 22.4.
constexpr int kFinishParts = 8192;
struct DistillArgs {
    Rows rows;
    int count;                         // rows in all
    const void *indices; int index_bits;
    const void *teacher; int teacher_type;
    int K;
    const int64_t *labels; int64_t ignore; int shift;
    float inv_tau, soft, hard;
    float soft_grad;                   // soft weight times tau
    int power;                         // tau where it is 2, 3 or 4
    int sum;                           // the gradient of the sum, not of the mean
    const int *live;                   // kCountBlocks partial counts of the live rows, or NULL: counted where they are needed
    const float *upstream;             // or NULL: 1
    char *grad;                        // [rows][V], or NULL
    double *part;                      // [workgroups][3]: hard loss, soft loss, live rows
};

__device__ __forceinline__ bool is_live(const DistillArgs &a, int64_t y) { return y != a.ignore && (uint64_t)y < (uint64_t)a.rows.V; }

// the label of row r, or -1 when the row is not live; -2 when there are no labels and every row is
__device__ __forceinline__ int row_label(const DistillArgs &a, int r) {
    if (!a.labels) return -2;
    int64_t y;
    if (a.shift) y = (r + 1) % a.rows.inner ? a.labels[r + 1] : (int64_t)0;       // the sequence moved left by one, 0 behind it
    else y = a.labels[r];
    return is_live(a, y) ? (int)y : -1;
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

// Live rows among those that this thread looks at, of `threads` threads.  Of shifted labels, the first of every sequence is
// nobody's and a 0 stands behind the last.
__device__ __forceinline__ int count_live(const DistillArgs &a, int first, int threads) {
    int n = 0;
    if (!a.labels) {
        for (int r = first; r < a.count; r += threads) ++n;
        return n;
    }
    for (int r = first; r < a.count; r += threads) n += is_live(a, a.labels[r]) ? 1 : 0;
    if (a.shift) {
        const int behind = is_live(a, 0) ? 1 : 0;
        for (int o = first; o < a.count / a.rows.inner; o += threads) n += behind - (is_live(a, a.labels[(int64_t)o * a.rows.inner]) ? 1 : 0);
    }
    return n;
}

// 1 / live rows (or 1) times the upstream gradient: from the count that a launch before this one has left, or (few rows) from
// the labels themselves.
__device__ __forceinline__ float over_live(const DistillArgs &a, int n) {
    const float s = a.upstream ? a.upstream[0] : 1.f;
    return a.sum ? s : n > 0 ? s / (float)n : 0.f;
}

// live rows, in kCountBlocks parts
__global__ __launch_bounds__(256) void distill_count_kernel(DistillArgs a, int *live) {
    __shared__ int s[4];
    int n = count_live(a, blockIdx.x * 256 + threadIdx.x, kCountBlocks * 256);
    n = wave_reduce(n, [](int x, int y) { return x + y; });
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) live[blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}

// Many workgroups' parts, added up to kCountBlocks of them before the last launch, which is one workgroup.
__global__ __launch_bounds__(256) void distill_add_kernel(const double *part, int n, double *sums) {
    __shared__ double s[3][4];
    double v[3] = {0.0, 0.0, 0.0};
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += kCountBlocks * 256) {
        v[0] += part[3 * (int64_t)i]; v[1] += part[3 * (int64_t)i + 1]; v[2] += part[3 * (int64_t)i + 2];
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        v[k] = wave_reduce(v[k], [](double x, double y) { return x + y; });
        if ((threadIdx.x & 63) == 0) s[k][threadIdx.x >> 6] = v[k];
    }
    __syncthreads();
    if (threadIdx.x < 3) sums[3 * blockIdx.x + threadIdx.x] = s[threadIdx.x][0] + s[threadIdx.x][1] + s[threadIdx.x][2] + s[threadIdx.x][3];
}

__global__ __launch_bounds__(1024) void distill_finish_kernel(const double *part, int n, float soft, float hard, int mean, float *loss, float *stats) {
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
        const double sum = (hard != 0.f ? (double)hard * v[0] : 0.0) + (soft != 0.f ? (double)soft * v[1] : 0.0);
        loss[0] = (float)(mean ? sum / (v[2] > 0.0 ? v[2] : 1.0) : sum);
        if (stats) { stats[0] = (float)sum; stats[1] = (float)v[2]; stats[2] = (float)v[0]; stats[3] = (float)v[1]; }
    }
}

// The compiler would keep the widened words, or their exponentials, from one use to the next (twice the registers for 16-bit
// words, and spills): behind this the pieces are new values to it.
template <int N>
__device__ __forceinline__ void hide_pieces(Raw (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i].w[0]), "+v"(x[i].w[1]), "+v"(x[i].w[2]), "+v"(x[i].w[3]));
}

template <int TPB>
struct RowShared {
    alignas(16) int index[kMaxTop];
    float share[kMaxTop];                        // e_k
    // words whose value is stored a second time, the label's last; and which of them lie in a wave's pieces
    int word[kMaxTop + 1];
    float value[kMaxTop + 1];
    uint16_t list[TPB / 64][kMaxTop + 1];
    int listed[TPB / 64];
    float top[2][TPB / 64], sums[4][TPB / 64], live[TPB / 64];
};

// Sums (or maxima) of N values over the workgroup: through a place of its own in LDS, so one barrier does.
template <int TPB, bool MAX, int N>
__device__ __forceinline__ void block_reduce(float (&place)[N][TPB / 64], float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = MAX ? wave_max(v[i]) : wave_sum(v[i]);
    if constexpr (TPB > 64) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) place[i][threadIdx.x >> 6] = v[i];
        }
    }
    lds_barrier();
    if constexpr (TPB > 64) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = place[i][0];
#pragma unroll
            for (int w = 1; w < TPB / 64; ++w) v[i] = MAX ? fmaxf(v[i], place[i][w]) : v[i] + place[i][w];
        }
    }
}

template <int TPB>
__device__ __forceinline__ float gradient_scale(const DistillArgs &a, RowShared<TPB> &sh) {
    if (a.sum) return over_live(a, 0);
    if (a.live) return over_live(a, (int)wave_sum((float)a.live[threadIdx.x & 63]));
    const float n = wave_sum((float)count_live(a, threadIdx.x, TPB));       // fewer than 2^23 rows: exact
    if ((threadIdx.x & 63) == 0) sh.live[threadIdx.x >> 6] = n;
    lds_barrier();
    float all = 0.f;
    for (int w = 0; w < TPB / 64; ++w) all += sh.live[w];
    return over_live(a, (int)all);
}

// How a word's two exponentials, exp((z - z_max) / tau) for the soft term and exp(z - z_max) for the hard one, are had.
// kOne: one of them is all there is (a single term, or tau = 1).  kPower: tau is 2, 3 or 4, the second is the first one's
// power.  kTwo: two.
enum Exponentials { kOne, kPower, kTwo };

// In powers of two and relative to the row's maximum.  NEAR: as 2^(a z + b), b = -a z_max rounded: one multiply-add a word;
// every exponential of a row is off by the same 2^delta, which the quotients do not show and the logarithms take off again.
// Otherwise (a maximum so far out that delta grows, a row of the type's lowest value say) the distance comes first.
template <int E, bool NEAR>
struct Exponents {
    float zmax, a0, a1, b0, b1;
    int power;
    // first: the first exponential.  other: the second one; kPower: what the first is multiplied by to give it.
    template <int N>
    __device__ __forceinline__ void operator()(const float (&z)[N], float (&first)[N], float (&other)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            first[i] = __builtin_amdgcn_exp2f(NEAR ? fmaf(z[i], a0, b0) : (z[i] - zmax) * a0);
            if constexpr (E == kTwo) other[i] = __builtin_amdgcn_exp2f(NEAR ? fmaf(z[i], a1, b1) : (z[i] - zmax) * a1);
            if constexpr (E == kPower) other[i] = first[i];
        }
        if constexpr (E == kPower) {
            if (power > 2) {
#pragma unroll
                for (int i = 0; i < N; ++i) other[i] *= first[i];
            }
            if (power > 3) {
#pragma unroll
                for (int i = 0; i < N; ++i) other[i] *= first[i];
            }
        }
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&z)[N], float &s0, float &s1) const {
        float first[N], other[N];
        (*this)(z, first, other);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s0 += first[i];
            if constexpr (E == kTwo) s1 += other[i];
            if constexpr (E == kPower) s1 = fmaf(first[i], other[i], s1);
        }
    }
    // c0 first exponential + c1 second one
    template <int N>
    __device__ __forceinline__ void mix(const float (&z)[N], float c0, float c1, float (&g)[N]) const {
        float first[N], other[N];
        (*this)(z, first, other);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (E == kOne) g[i] = c0 * first[i];
            if constexpr (E == kTwo) g[i] = fmaf(c1, other[i], c0 * first[i]);
            if constexpr (E == kPower) g[i] = first[i] * fmaf(c1, other[i], c0);
        }
    }
};

// Longer rows (group_of, below), a workgroup per row.
//
// NR > 0: the row stays in NR pieces per thread.
// NR = 0: the row is read a second time for the gradient, and its maximum and sums come from one pass in which a thread
// rescales its sums when its maximum grows (rows longer than the registers hold, and the loss alone).
//
// The words that the teacher or the label names get their value a second time, from the wave that has stored their piece:
// a wave's stores to one place stay in order, so nothing waits for the row.
template <class T, int TPB, int NR, int E, bool GRAD>
__global__ __launch_bounds__(TPB) __attribute__((amdgpu_waves_per_eu(4))) void distill_row_kernel(DistillArgs a) {
    __shared__ RowShared<TPB> sh;
    constexpr int NK = TPB >= kMaxTop ? 1 : kMaxTop / TPB;      // teacher entries per thread
    constexpr int N = T::vec;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, V = a.rows.V;
    const int pieces = V / N, rest = V - pieces * N;            // whole 16-byte pieces, and words behind them: one a thread
    const int r = blockIdx.x, label = row_label(a, r);
    double *part = a.part + 3 * (int64_t)r;
    char *out = GRAD ? a.grad + (int64_t)r * V * T::bytes : nullptr;
    auto store = [&](char *to, const Raw &w) { store16<T, NR == 0>(to, w); };
    if (label == -1) {                 // not live: neither its words nor its teacher's are read
        if constexpr (GRAD) {
            for (int p = tid; p < pieces; p += TPB) store(out + (int64_t)p * 16, Raw{{0, 0, 0, 0}});
            if (tid < rest) store1<T>(out, pieces * N + tid, 0.f);
        }
        if (tid < 3) part[tid] = 0.0;
        return;
    }
    const char *row = a.rows.row(r);
    // piece i of this thread begins at byte 16 (tid + i TPB): a uniform address per i and one offset for all of them
    const uint32_t at16 = (uint32_t)tid * 16;
    auto has = [&](int i) { return tid < pieces - i * TPB; };
    Raw x[NR ? NR : 1];
#pragma unroll
    for (int i = 0; i < NR; ++i)
        if (has(i)) x[i] = load16<T, true>(row + i * TPB * 16 + at16);
    const float last[1] = {tid < rest ? load1<T>(row, pieces * N + tid) : -INFINITY};
    auto hide = [&]() { if constexpr (NR > 0) hide_pieces(x); };
    auto widen = [](const Raw &w, float (&z)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = element<T>(w, e);
    };

    int idx[NK];
    float t[NK], zk[NK];
    float top[2] = {last[0], -INFINITY};          // of the row, of the teacher's entries
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        const int k = tid + j * TPB;
        idx[j] = -1; t[j] = -INFINITY; zk[j] = 0.f;
        if (k < a.K) {
            const int64_t at = (int64_t)r * a.K + k;
            idx[j] = teacher_index(a, at);
            if (idx[j] >= 0) { t[j] = teacher_value(a, at); zk[j] = load1<T>(row, idx[j]); }
        }
        if (GRAD && k < kMaxTop) sh.index[k] = idx[j];
        top[1] = fmaxf(top[1], t[j]);
    }
    if (GRAD && tid < TPB / 64) sh.listed[tid] = 0;
    const float zy = label >= 0 ? load1<T>(row, label) : 0.f;

    const float a0 = (E != kOne || a.soft != 0.f ? a.inv_tau : 1.f) * kLog2e, a1 = kLog2e;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};         // sum of the first exponential, of the second, A, B
    if constexpr (NR > 0) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (has(i)) {
#pragma unroll
                for (int e = 0; e < N; ++e) top[0] = fmaxf(top[0], element<T>(x[i], e));
            }
    } else {
        float ref = fmaxf(last[0], -FLT_MAX);
        Exponents<E, false> ex{ref, a0, a1, 0.f, 0.f, a.power};
        auto grow = [&](float m) {
            if (m > ref) {
                const float d = ref - m;
                sums[0] *= __builtin_amdgcn_exp2f(d * a0);
                if constexpr (E != kOne) sums[1] *= __builtin_amdgcn_exp2f(d * a1);
                ref = m;
            }
            ex.zmax = ref;
        };
        auto add = [&](const Raw &w) {
            float z[N];
            widen(w, z);
            ex.add(z, sums[0], sums[1]);
        };
        constexpr int U = 4;
        int p = tid;
        for (; p + (U - 1) * TPB < pieces; p += U * TPB) {
            Raw w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = load16<T, !GRAD>(row + (int64_t)(p + u * TPB) * 16);
            float m = ref;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) m = fmaxf(m, element<T>(w[u], e));
            grow(m);
#pragma unroll
            for (int u = 0; u < U; ++u) add(w[u]);
        }
        for (; p < pieces; p += TPB) {
            const Raw w = load16<T>(row + (int64_t)p * 16);
            float m = ref;
#pragma unroll
            for (int e = 0; e < N; ++e) m = fmaxf(m, element<T>(w, e));
            grow(m);
            add(w);
        }
        top[0] = ref;
    }
    const float mine = top[0];
    block_reduce<TPB, true>(sh.top, top);
    hide();
    const float zmax = top[0], tmax = top[1];
    const float b0 = -zmax * a0, b1 = -zmax * a1;
    const bool near = NR > 0 && fabsf(b0) < 1048576.f && fabsf(b1) < 1048576.f;       // delta below 2^-4 then
    const Exponents<E, true> fast{zmax, a0, a1, b0, b1, a.power};
    const Exponents<E, false> plain{zmax, a0, a1, b0, b1, a.power};
    if (near) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (has(i)) {
                float z[N];
                widen(x[i], z);
                fast.add(z, sums[0], sums[1]);
            }
        if (tid < rest) fast.add(last, sums[0], sums[1]);
    } else {
        if constexpr (NR > 0) {
            for (int p = tid; p < pieces; p += TPB) {
                float z[N];
                widen(load16<T>(row + (int64_t)p * 16), z);
                plain.add(z, sums[0], sums[1]);
            }
        } else {
            sums[0] *= __builtin_amdgcn_exp2f((mine - zmax) * a0);
            if constexpr (E != kOne) sums[1] *= __builtin_amdgcn_exp2f((mine - zmax) * a1);
        }
        if (tid < rest) plain.add(last, sums[0], sums[1]);
    }
    float share[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        const int k = tid + j * TPB;
        const float d = t[j] - tmax;
        share[j] = idx[j] >= 0 && t[j] != -INFINITY ? __builtin_amdgcn_exp2f(d * a0) : 0.f;
        if (share[j] != 0.f) {
            sums[2] += share[j];
            sums[3] += share[j] * (d - (zk[j] - zmax));
        }
        if (GRAD && k < a.K) sh.share[k] = share[j];
    }
    block_reduce<TPB, false>(sh.sums, sums);
    const float s0 = sums[0], s1 = E != kOne ? sums[1] : sums[0], A = sums[2], B = sums[3];
    if (tid == 0) {
        // the row's sums without the common factor 2^delta (its power in the second one)
        const float off0 = near ? fmaf(zmax, a0, b0) * 0.6931471805599453f : 0.f;
        const float off1 = E == kPower ? off0 * (float)a.power : E == kTwo && near ? fmaf(zmax, a1, b1) * 0.6931471805599453f : off0;
        part[0] = a.hard != 0.f ? (double)(logf(s1) - off1 - (zy - zmax)) : 0.0;
        part[1] = a.soft != 0.f && A != 0.f ? (double)B / A * (a0 * 0.6931471805599453) + log((double)s0 / A) - off0 : 0.0;
        part[2] = 1.0;
    }
    if constexpr (GRAD) {
        hide();
        const float scale = gradient_scale<TPB>(a, sh);
        const float soft = a.soft != 0.f && A != 0.f ? a.soft_grad * scale : 0.f, hard = a.hard != 0.f ? a.hard * scale : 0.f;
        const float c0 = E != kOne ? soft / s0 : (soft + hard) / s0, c1 = E != kOne ? hard / s1 : 0.f;
        auto density = [&](float v) {
            const float z[1] = {v};
            float g[1];
            if (near) fast.mix(z, c0, c1, g);
            else plain.mix(z, c0, c1, g);
            return g[0];
        };
        // the named words' values; an index that comes twice is left to its first entry, with both shares
        auto name = [&](int k, int v, float value) {
            const int p = v / N, owner = (p < pieces ? p & (TPB - 1) : v - pieces * N) >> 6;
            sh.word[k] = v;
            sh.value[k] = value;
            sh.list[owner][atomicAdd(&sh.listed[owner], 1)] = (uint16_t)k;
        };
        const float soft_share = A != 0.f ? soft / A : 0.f;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const int k = tid + j * TPB;
            if (idx[j] < 0) continue;
            int same = 0;
            for (int i = 0; i < a.K; i += 4) {
                const int4 q = *(const int4 *)&sh.index[i];       // behind K: -1
                same += (q.x == idx[j]) + (q.y == idx[j]) + (q.z == idx[j]) + (q.w == idx[j]);
            }
            float named = share[j];
            bool first = true;
            if (same > 1) {
                named = 0.f;
                for (int i = 0; i < a.K; ++i)
                    if (sh.index[i] == idx[j]) { first = first && i >= k; named += sh.share[i]; }
            }
            if (first) name(k, idx[j], density(zk[j]) - soft_share * named - (idx[j] == label ? hard : 0.f));
        }
        if (wave == TPB / 64 - 1 && label >= 0 && hard != 0.f) {
            bool named = false;
            for (int i = lane; i < a.K; i += 64) named = named || sh.index[i] == label;
            if (!__ballot(named) && lane == 0) name(kMaxTop, label, density(zy) - hard);
        }
        if (near) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
                if (has(i)) {
                    float z[N], g[N];
                    widen(x[i], z);
                    fast.mix(z, c0, c1, g);
                    store(out + i * TPB * 16 + at16, pack<T>(g));
                }
        } else {
            constexpr int U = 4;
            auto put = [&](const Raw &w, int p) {
                float z[N], g[N];
                widen(w, z);
                plain.mix(z, c0, c1, g);
                store(out + (int64_t)p * 16, pack<T>(g));
            };
            int p = tid;
            if constexpr (NR == 0) {
                for (; p + (U - 1) * TPB < pieces; p += U * TPB) {
                    Raw w[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) w[u] = load16<T, true>(row + (int64_t)(p + u * TPB) * 16);
#pragma unroll
                    for (int u = 0; u < U; ++u) put(w[u], p + u * TPB);
                }
            }
            for (; p < pieces; p += TPB) put(load16<T>(row + (int64_t)p * 16), p);
        }
        if (tid < rest) store1<T>(out, pieces * N + tid, density(last[0]));
        lds_barrier();
        for (int i = lane; i < sh.listed[wave]; i += 64) {
            const int k = sh.list[wave][i];
            store1<T>(out, sh.word[k], sh.value[k]);
        }
    }
}

// Short rows: L lanes per row, P pieces a lane, 256 / L rows in a workgroup; the reductions stay within a row's lanes and no
// row waits for another.  The teacher's entries (word, share, the student's logit) lie in LDS; a row's belong to its wave,
// whose LDS accesses are in order.
template <class T, int L, int P, bool GRAD>
__global__ __launch_bounds__(256) void distill_group_kernel(DistillArgs a, int stride) {
    extern __shared__ int4 entries[];
    constexpr int R = 256 / L, N = T::vec;
    __shared__ double s_linear[2][R], s_factor[2][R];
    __shared__ int s_rows[R], s_live[4];
    const int slot = threadIdx.x / L, lane = threadIdx.x & (L - 1), r = blockIdx.x * R + slot, V = a.rows.V, K = a.K;
    const int full = V / N, rest = V - full * N;                // whole 16-byte pieces, and words behind them
    int *index = (int *)entries + slot * stride;                // [R][stride] each
    float *share = (float *)index + R * stride, *words = share + R * stride;
    const int label = r < a.count ? row_label(a, r) : -1;
    const bool live = label != -1;
    const char *row = a.rows.row(r < a.count ? r : 0);
    constexpr uint32_t none = __is_same(T, TypeF32) ? 0xff800000u : __is_same(T, TypeBF16) ? 0xff80ff80u : 0xfc00fc00u;      // -inf
    Raw x[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int p = lane + i * L;
        if (live && p < full) x[i] = load16<T, true>(row + (int64_t)p * 16);
        else if (live && p == full && rest) x[i] = load_tail<T>(row, p * N, V);
        else x[i] = Raw{{none, none, none, none}};
    }
    const float zy = label >= 0 ? load1<T>(row, label) : 0.f;
    float tmax = -INFINITY, zmax = -INFINITY;
    for (int k = lane; k < stride; k += L) {
        int v = -1;
        float t = -INFINITY, z = 0.f;
        if (live && k < K) {
            const int64_t at = (int64_t)r * K + k;
            v = teacher_index(a, at);
            if (v >= 0) { t = teacher_value(a, at); z = load1<T>(row, v); }
        }
        index[k] = v; share[k] = t; words[k] = z;
        tmax = fmaxf(tmax, t);
    }
    auto widen = [](const Raw &w, float (&z)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = element<T>(w, e);
    };
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) zmax = fmaxf(zmax, element<T>(x[i], e));
    auto larger = [](float u, float v) { return fmaxf(u, v); };
    auto plus = [](double u, double v) { return u + v; };
    zmax = group_reduce<L>(zmax, larger);
    tmax = group_reduce<L>(tmax, larger);

    const bool soft_on = a.soft != 0.f, hard_on = a.hard != 0.f, two = soft_on && hard_on && a.inv_tau != 1.f;
    const float a0 = (soft_on ? a.inv_tau : 1.f) * kLog2e;
    // the soft term's exponentials, and the hard one's where they differ (`two`)
    auto exponentials = [&](const float (&z)[N], float (&first)[N], float (&second)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) first[e] = __builtin_amdgcn_exp2f((z[e] - zmax) * a0);
        if (!two) return;
        if (a.power) {
#pragma unroll
            for (int e = 0; e < N; ++e) second[e] = first[e] * first[e];
            if (a.power > 2) {
#pragma unroll
                for (int e = 0; e < N; ++e) second[e] *= a.power > 3 ? second[e] : first[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) second[e] = __builtin_amdgcn_exp2f((z[e] - zmax) * kLog2e);
        }
    };
    // in 64 bits: where the student nearly agrees with a teacher that names all words, little is left of these sums, and their
    // roundings would be most of its error
    double sum0 = 0.0, sum1 = 0.0, sumA = 0.0, sumB = 0.0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        float z[N], first[N], second[N];
        widen(x[i], z);
        exponentials(z, first, second);
#pragma unroll
        for (int e = 0; e < N; ++e) sum0 += (double)first[e];
        if (two) {
#pragma unroll
            for (int e = 0; e < N; ++e) sum1 += (double)second[e];
        }
    }
    for (int k = lane; k < K; k += L) {
        const float t = share[k], d = t - tmax;
        const float e = index[k] >= 0 && t != -INFINITY ? __builtin_amdgcn_exp2f(d * a0) : 0.f;
        if (e != 0.f) { sumA += (double)e; sumB += (double)e * (double)(d - (words[k] - zmax)); }
        share[k] = e;
    }
    sum0 = group_reduce<L>(sum0, plus);
    sum1 = two ? group_reduce<L>(sum1, plus) : sum0;
    sumA = group_reduce<L>(sumA, plus);
    sumB = group_reduce<L>(sumB, plus);
    const float s0 = (float)sum0, s1 = (float)sum1, A = (float)sumA;
    if constexpr (GRAD) {
        int n = 0;
        if (!a.sum) n = a.live ? a.live[threadIdx.x & 63] : count_live(a, threadIdx.x, 256);
        n = wave_reduce(n, [](int u, int v) { return u + v; });
        if (!a.sum && !a.live) {
            if ((threadIdx.x & 63) == 0) s_live[threadIdx.x >> 6] = n;
            __syncthreads();
            n = s_live[0] + s_live[1] + s_live[2] + s_live[3];
        }
        const float scale = over_live(a, n);
        const float soft = soft_on && A != 0.f ? a.soft_grad * scale : 0.f, hard = hard_on ? a.hard * scale : 0.f;
        const float c0 = two ? soft / s0 : (soft + hard) / s0, c1 = two ? hard / s1 : 0.f;
        auto mix = [&](const float (&z)[N], float (&g)[N]) {
            float first[N], second[N];
            exponentials(z, first, second);
#pragma unroll
            for (int e = 0; e < N; ++e) g[e] = two ? fmaf(c1, second[e], c0 * first[e]) : c0 * first[e];
        };
        char *out = a.grad + (int64_t)r * V * T::bytes;
        hide_pieces(x);
        if (r < a.count) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int p = lane + i * L;
                float z[N], g[N];
                widen(x[i], z);
                mix(z, g);
#pragma unroll
                for (int e = 0; e < N; ++e) g[e] = live ? g[e] : 0.f;
                if (p < full) store16<T>(out + (int64_t)p * 16, pack<T>(g));
                else if (p == full) {
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (e < rest) store1<T>(out, p * N + e, g[e]);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // the words that the teacher or the label names, a second time, by the wave that has stored them
        auto density = [&](float v) {
            const float d = v - zmax, first = __builtin_amdgcn_exp2f(d * a0);
            return two ? fmaf(c1, __builtin_amdgcn_exp2f(d * kLog2e), c0 * first) : c0 * first;
        };
        const float soft_share = A != 0.f ? soft / A : 0.f;
        float named_label = 0.f;
        for (int k = lane; k < K; k += L) {
            const int v = index[k];
            if (v < 0) continue;
            int same = 0;
            for (int i = 0; i < K; i += 4) {
                const int4 q = *(const int4 *)&index[i];        // behind K: -1
                same += (q.x == v) + (q.y == v) + (q.z == v) + (q.w == v);
            }
            float named = share[k];
            bool first = true;
            if (same > 1) {                                     // left to its first entry, with all of the shares
                named = 0.f;
                for (int i = 0; i < K; ++i)
                    if (index[i] == v) { first = first && i >= k; named += share[i]; }
            }
            if (v == label) named_label = 1.f;
            if (first) store1<T>(out, v, density(words[k]) - soft_share * named - (v == label ? hard : 0.f));
        }
        if (hard_on) {
            named_label = group_reduce<L>(named_label, larger);
            if (lane == 0 && label >= 0 && named_label == 0.f) store1<T>(out, label, density(zy) - hard);
        }
    }
    // the rows' losses are  linear + log(factor)  each; one logarithm takes the product of a workgroup's factors (each within
    // 2^-8 .. 2^10, 64 of them at most)
    if (lane == 0) {
        const bool soft = live && soft_on && A != 0.f, hard = live && hard_on;
        const double inverse = 1.0 / (soft ? sumA : 1.0);
        s_linear[0][slot] = hard ? -(double)(zy - zmax) : 0.0;
        s_factor[0][slot] = hard ? sum1 : 1.0;
        s_linear[1][slot] = soft ? sumB * inverse * (a0 * 0.6931471805599453) : 0.0;
        s_factor[1][slot] = soft ? sum0 * inverse : 1.0;
        s_rows[slot] = live ? 1 : 0;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int i = threadIdx.x;
    double linear[2], factor[2];
    int rows = i < R ? s_rows[i] : 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) { linear[k] = i < R ? s_linear[k][i] : 0.0; factor[k] = i < R ? s_factor[k][i] : 1.0; }
    auto over_rows = [](auto v, auto op) {
        v = group_reduce<16>(v, op);
#pragma unroll
        for (int d = 16; d < R; d <<= 1) v = op(v, __shfl_xor(v, d));
        return v;
    };
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        linear[k] = over_rows(linear[k], plus);
        factor[k] = over_rows(factor[k], [](double u, double v) { return u * v; });
    }
    rows = over_rows(rows, [](int u, int v) { return u + v; });
    if (i < 3) a.part[3 * (int64_t)blockIdx.x + i] = i == 2 ? (double)rows : (i ? linear[1] : linear[0]) + log(i ? factor[1] : factor[0]);
}

// Rows of up to 8 pieces for each of 16 lanes go to groups of lanes: what a row costs whatever its length (reductions, the
// teacher's entries, quotients: about 400 instructions of a wave) is then shared by 4 to 16 rows, where a workgroup of one wave
// per row spends it on each.  262144 rows, loss and gradient / loss alone, against a wave per row: 100 words of float 94 / 53 for
// 275 / 134 us, 200: 133 / 72 for 296 / 146, 500: 282 / 129 for 379 / 182; of bfloat16 120: 94 / 55 for 300 / 174, 500: 198 / 90
// for 362 / 233; 32768 rows of 1000: 58 / 27 for 62 / 35.  (Against a word per lane: 9 words 32 / 17 for 55 / 37, 40 words 77 / 45
// for 175 / 134.  Sums in 32 bits would be 3 to 10 % faster, a logarithm per row up to a third slower.)  Issue binds them up to some 200
// words: 262144 rows of 40 words take 653 VALU instructions a wave of 4 rows, 1.00 per SIMD and four cycles, of 100 words 696 and
// 0.88; the bytes beyond (500 words of float: 3.7 TB/s).
constexpr int kGroupPieces = 8, kGroupLds = 48 * 1024;
struct Group { int L, P, stride; };
bool grouped(const gscan_rows &rows) { return cdiv(rows.V, rows.type == GSCAN_F32 ? 4 : 8) <= 16 * kGroupPieces; }
Group group_of(const gscan_rows &rows, int K) {
    const int pieces = cdiv(rows.V, rows.type == GSCAN_F32 ? 4 : 8), stride = (K + 3) & ~3;
    int L = pieces <= 4 ? 4 : pieces <= 8 ? 8 : 16;
    while (256 / L * stride * 12 > kGroupLds) L *= 2;           // 16 lanes hold any number of entries
    return Group{L, cdiv(pieces, L), stride};
}
int part_blocks(const gscan_rows &rows, int K) {
    const int64_t n = rows.outer * rows.inner;
    return grouped(rows) ? cdiv(n, 256 / group_of(rows, K).L) : (int)n;
}

template <class T, int L, int P>
int launch_group(const DistillArgs &a, int stride, hipStream_t stream) {
    const dim3 grid(cdiv(a.count, 256 / L)), block(256);
    const size_t lds = (size_t)(256 / L) * stride * 12;
    if (a.grad) hipLaunchKernelGGL((distill_group_kernel<T, L, P, true>), grid, block, lds, stream, a, stride);
    else hipLaunchKernelGGL((distill_group_kernel<T, L, P, false>), grid, block, lds, stream, a, stride);
    GSCAN_LAUNCHED("distill_group_kernel");
    return 0;
}

template <class T, int TPB, int NR, bool GRAD>
int launch_row(const DistillArgs &a, hipStream_t stream) {
    const dim3 grid(a.count), block(TPB);
    const bool two = a.hard != 0.f && a.soft != 0.f && a.inv_tau != 1.f;
    if (two && a.power) hipLaunchKernelGGL((distill_row_kernel<T, TPB, NR, kPower, GRAD>), grid, block, 0, stream, a);
    else if (two) hipLaunchKernelGGL((distill_row_kernel<T, TPB, NR, kTwo, GRAD>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((distill_row_kernel<T, TPB, NR, kOne, GRAD>), grid, block, 0, stream, a);
    GSCAN_LAUNCHED("distill_row_kernel");
    return 0;
}

template <class T>
int launch_type(const DistillArgs &a, const gscan_rows &rows, hipStream_t stream) {
    const int V = a.rows.V;
    if (grouped(rows)) {
        const Group g = group_of(rows, a.K);
        if (g.L == 4) return launch_group<T, 4, 1>(a, g.stride, stream);
        if (g.L == 8) return launch_group<T, 8, 1>(a, g.stride, stream);
        if (g.P == 1) return launch_group<T, 16, 1>(a, g.stride, stream);
        if (g.P == 2) return launch_group<T, 16, 2>(a, g.stride, stream);
        if (g.P <= 4) return launch_group<T, 16, 4>(a, g.stride, stream);
        return launch_group<T, 16, 8>(a, g.stride, stream);
    }
    const int pieces = V / T::vec;
    // Registers hold a row of up to 128 KB: 8 pieces a thread while 512 threads do (32000 bfloat16 words: 104 us for 459 MB, 4.4
    // TB/s; 256 threads of 16 pieces 134 for 124, 1024 of 4 171), then 16.  Longer ones are streamed twice, the gradient past the
    // caches (4096 rows of 131072 words, 1.9 GB with a quarter of them not live: 430 us; held by 1024 threads 540).  The loss alone is
    // one streamed pass (2000 rows of 65537 half words: 51 us).
    if (!a.grad) {
        if (pieces <= 64 * 8) return launch_row<T, 64, 0, false>(a, stream);
        return launch_row<T, 512, 0, false>(a, stream);
    }
    if (pieces <= 64 * 8) return launch_row<T, 64, 8, true>(a, stream);
    if (pieces <= 256 * 8) return launch_row<T, 256, 8, true>(a, stream);
    if (pieces <= 512 * 8) return launch_row<T, 512, 8, true>(a, stream);
    if (pieces <= 512 * 16) return launch_row<T, 512, 16, true>(a, stream);
    return launch_row<T, 512, 0, true>(a, stream);
}
}  // namespace

size_t distillation_workspace(const gscan_rows &rows) {
    return kCountBlocks * (sizeof(int) + 3 * sizeof(double)) + (size_t)(grouped(rows) ? cdiv(rows.outer * rows.inner, 16) : rows.outer * rows.inner) * 3 * sizeof(double);
}

int distillation_loss(const gscan_rows &rows, const gscan_distillation &t, const float *upstream, void *grad, float *loss,
                      float *stats, void *workspace, size_t bytes, hipStream_t stream) {
    GSCAN_CHECK(loss || (grad && !stats), "distillation_loss: loss is NULL");
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
    a.power = t.temperature == 2.f ? 2 : t.temperature == 3.f ? 3 : t.temperature == 4.f ? 4 : 0;
    a.upstream = upstream; a.grad = (char *)grad;
    double *sums = (double *)(live + kCountBlocks);
    a.part = sums + 3 * kCountBlocks;
    a.sum = t.sum_reduction != 0;
    if (grad && !a.sum && a.count > (grouped(rows) ? kCountThere : kCountThereLong)) {       // the gradient of a mean needs the number of live rows first
        a.live = live;
        hipLaunchKernelGGL(distill_count_kernel, dim3(kCountBlocks), dim3(256), 0, stream, a, live);
        GSCAN_LAUNCHED("distill_count_kernel");
    }
    const int type = rows.type;
    TRY_RC(type == GSCAN_F32    ? launch_type<TypeF32>(a, rows, stream)
           : type == GSCAN_BF16 ? launch_type<TypeBF16>(a, rows, stream)
                                : launch_type<TypeF16>(a, rows, stream));
    if (!loss) return 0;
    const float tau2 = t.temperature * t.temperature;
    const double *part = a.part;
    int parts = part_blocks(rows, t.K);
    if (parts > kFinishParts) {
        hipLaunchKernelGGL(distill_add_kernel, dim3(kCountBlocks), dim3(256), 0, stream, part, parts, sums);
        GSCAN_LAUNCHED("distill_add_kernel");
        part = sums;
        parts = kCountBlocks;
    }
    hipLaunchKernelGGL(distill_finish_kernel, dim3(1), dim3(1024), 0, stream, part, parts, t.soft_weight * tau2,
                       t.hard_weight, t.sum_reduction ? 0 : 1, loss, stats);
    GSCAN_LAUNCHED("distill_finish_kernel");
    return 0;
}

}  // namespace gscan
