// The K best words of every row of logits, in order, with the row's log-sum-exp: what a teacher leaves for its student
// (distill.hip) and what a beam search looks at in a step (beam.hip).  Order: value descending, index ascending; a NaN counts
// as -inf.
//
// One pass over the row, then a few per mille of it a second time: 4 TPB groups of a row's 16-byte pieces keep one maximum
// each.  At least K words are >= the K-th largest of these maxima, so it bounds the K-th largest word from below, and a group
// whose maximum is below the bound holds none of the K: only the other groups' pieces are read again, and what is >= the bound
// (little more than K words unless many are equal) is ranked in LDS by counting.  Exact for any input: where the words >= the
// bound do not fit the list, words above it and, in index order, words equal to it are taken apart, and if even the words
// above it do not fit (a row laid out against this grouping), a radix selection over the row finds the K-th key.
#include <cstddef>

#include "logits.h"

namespace gscan {

namespace {
constexpr int kCap = 1024;         // candidates in LDS: at least 4 kMaxTop

struct TopArgs {
    Rows rows;
    int K, splits, chunk;
    void *values; int32_t *indices; float *lse;      // splits == 1
    uint64_t *keys; LsePart *parts;                  // otherwise (and for the beam step)
    const uint8_t *finished; const float *scores;    // beam step: a row that is finished or has no score is left out
};

// Words of a row (or of a part of it), 16 bytes at a time.
template <class T>
struct WordSource {
    static constexpr int vec = T::vec;
    const char *row;      // of the whole row
    int first, n;         // the part: words [first, first + n), first a multiple of vec
    __device__ __forceinline__ int pieces() const { return (n + vec - 1) / vec; }
    __device__ __forceinline__ Raw load(int p) const { return load_group<T>(row + (int64_t)first * T::bytes, p, n); }
    __device__ __forceinline__ uint64_t entry(const Raw &r, int p, int e) const {       // 0: behind the end
        const int i = p * vec + e;
        return i < n ? pair_key(order_key(element<T>(r, e)), first + i) : 0ull;
    }
    __device__ __forceinline__ uint64_t at(int i) const {
        return pair_key(order_key(load1<T>(row, first + i)), first + i);
    }
};
// Entries that chunks of a row have left, one at a time (0: none).
struct EntrySource {
    static constexpr int vec = 1;
    const uint64_t *list;
    int n;
    __device__ __forceinline__ int pieces() const { return n; }
    __device__ __forceinline__ uint64_t load(int p) const { return list[p]; }
    __device__ __forceinline__ uint64_t entry(uint64_t r, int, int) const { return r; }
    __device__ __forceinline__ uint64_t at(int i) const { return list[i]; }
};

template <int TPB>
struct TopShared {
    alignas(16) uint64_t cand[kCap + 2];
    uint32_t keys[4 * TPB];         // the groups' maxima; the radix selection's histogram
    uint32_t thread_keys[TPB];
    uint16_t hit[4 * TPB];          // groups to read again
    uint32_t bound;
    int hits, count, above;
    int wave_count[TPB / 64];
    double sum[TPB / 64];
    float ref[TPB / 64];
};

// Reads the pieces of the groups on the list again and puts the entries whose key is > bound (or >= it) on the list of
// candidates; returns how many there are, which may be more than fit.
template <int TPB, class S>
__device__ __forceinline__ int collect(const S &src, TopShared<TPB> &sh, uint32_t bound, bool equal) {
    const int tid = threadIdx.x, hits = sh.hits, pieces = src.pieces();
    const int per = (pieces + 4 * TPB - 1) / (4 * TPB);
    const int items = hits * per;
    for (int it = tid; it < items; it += TPB) {
        const int h = it / per, p = sh.hit[h] + (it - h * per) * (4 * TPB);
        if (p >= pieces) continue;
        const auto raw = src.load(p);
#pragma unroll
        for (int e = 0; e < S::vec; ++e) {
            const uint64_t x = src.entry(raw, p, e);
            const uint32_t k = (uint32_t)(x >> 32);
            if (k > bound || (equal && k == bound && k)) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kCap) sh.cand[at] = x;
            }
        }
    }
    __syncthreads();
    return sh.count;
}

// The first `want` entries, in index order, whose key is `key`, behind the `at` candidates that are there.
template <int TPB, class S>
__device__ void collect_equal(const S &src, TopShared<TPB> &sh, uint32_t key, int at, int want) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, words = src.pieces() * S::vec;
    int found = 0;
    for (int base = 0; base < words && found < want; base += TPB) {
        const int i = base + tid;
        const uint64_t x = i < src.n ? src.at(i) : 0ull;
        const bool is = x && (uint32_t)(x >> 32) == key;
        const unsigned long long b = __ballot(is);
        if (lane == 0) sh.wave_count[wave] = __popcll(b);
        __syncthreads();
        int before = found, total = 0;
        for (int w = 0; w < TPB / 64; ++w) {
            if (w < wave) before += sh.wave_count[w];
            total += sh.wave_count[w];
        }
        const int mine = before + __popcll(b & ((1ull << lane) - 1));
        if (is && mine < want) sh.cand[at + mine] = x;
        found += total;
        __syncthreads();
    }
}

// The K-th largest key of the whole source by radix selection (eight bits a pass); returns how many entries equal to it
// belong to the K.  Entered with more than K entries.
template <int TPB, class S>
__device__ int radix_select(const S &src, TopShared<TPB> &sh, int K, uint32_t *key) {
    const int tid = threadIdx.x, pieces = src.pieces();
    uint32_t prefix = 0;
    int need = K;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += TPB) sh.keys[i] = 0;
        __syncthreads();
        for (int p = tid; p < pieces; p += TPB) {
            const auto raw = src.load(p);
#pragma unroll
            for (int e = 0; e < S::vec; ++e) {
                const uint32_t k = (uint32_t)(src.entry(raw, p, e) >> 32);
                if (k && (shift == 24 || (k >> (shift + 8)) == prefix)) atomicAdd(&sh.keys[(k >> shift) & 255], 1u);
            }
        }
        __syncthreads();
        if (tid < 64) {       // lane l holds the bins 255 - 4l .. 252 - 4l
            int c[4], mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) { c[i] = (int)sh.keys[255 - 4 * tid - i]; mine += c[i]; }
            int upto = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(upto, d); if (tid >= d) upto += o; }
            int before = upto - mine;
            if (before < need && upto >= need) {
                for (int i = 0; i < 4; ++i) {
                    if (before + c[i] >= need) { sh.bound = (uint32_t)(255 - 4 * tid - i); sh.above = need - before; break; }
                    before += c[i];
                }
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | sh.bound;
        need = sh.above;
        __syncthreads();
    }
    *key = prefix;
    return need;
}

// With the groups' maxima in sh.keys (and, for a small K, the threads' maxima over their four groups in sh.thread_keys):
// leaves candidates that hold the K best entries in sh.cand and returns their number.  `scan(bound)` puts the entries >= bound
// on the list without reading again, where it can.
template <int TPB, class S, class F>
__device__ int find_candidates(const S &src, TopShared<TPB> &sh, int K, F scan) {
    constexpr int G = 4 * TPB;
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid < 64) {
        // K of TPB threads' maxima bound nearly as well as K of four times as many, for a quarter of the counting, while K is
        // no more than a quarter of them
        const uint32_t b = 4 * K <= TPB ? kth_bound<TPB / 64>(sh.thread_keys, TPB, K, tid) : kth_bound<G / 64>(sh.keys, G, K, tid);
        if (tid == 0) { sh.bound = b; sh.hits = 0; sh.count = 0; }
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    if constexpr (!__is_same(F, std::nullptr_t)) {
        scan(bound);
        __syncthreads();
        if (sh.count <= kCap) return sh.count;
        __syncthreads();
        if (tid == 0) sh.count = 0;
    }
    for (int g = tid; g < G; g += TPB)
        if (sh.keys[g] >= bound && sh.keys[g]) sh.hit[atomicAdd(&sh.hits, 1)] = (uint16_t)g;
    __syncthreads();
    int n;
    if constexpr (__is_same(F, std::nullptr_t)) {
        n = collect<TPB>(src, sh, bound, true);
        if (n <= kCap) return n;
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
    }
    n = collect<TPB>(src, sh, bound, false);
    if (n >= K && n <= kCap) return n;
    if (n < K) {
        collect_equal<TPB>(src, sh, bound, n, K - n);
        return K;
    }
    __syncthreads();
    uint32_t key;
    const int equal = radix_select<TPB>(src, sh, K, &key);
    // every group may hold entries above the K-th key: all of them are read again
    if (tid == 0) { sh.hits = G; sh.count = 0; }
    for (int g = tid; g < G; g += TPB) sh.hit[g] = (uint16_t)g;
    __syncthreads();
    n = collect<TPB>(src, sh, key, false);
    collect_equal<TPB>(src, sh, key, n, equal);
    return K;
}

// Every candidate's place is the number of candidates before it; `put(place, entry)` for the first K of them.
template <int TPB, class F>
__device__ __forceinline__ void rank_candidates(TopShared<TPB> &sh, int n, int K, F put) {
    const int even = (n + 1) & ~1;
    if (threadIdx.x == 0 && even > n) sh.cand[n] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += TPB) {
        const uint64_t x = sh.cand[i];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < even; j += 2) {
            const ulonglong2 q = *(const ulonglong2 *)&sh.cand[j];
            place += (q.x > x ? 1 : 0) + (q.y > x ? 1 : 0);
        }
        if (place < K) put(place, x);
    }
}

template <class T>
__device__ __forceinline__ void put_out(const TopArgs &a, int64_t at, uint64_t x) {
    store1<T>((char *)a.values, at, key_value((uint32_t)(x >> 32)));
    a.indices[at] = (int32_t)~(uint32_t)x;
}

// One workgroup per row, or per chunk of a row.  HELD: a row (chunk) of at most four pieces a thread, which stay in registers:
// nothing is read again.
template <class T, int TPB, bool LSE, bool HELD>
__global__ __launch_bounds__(TPB) void top_row_kernel(TopArgs a) {
    __shared__ TopShared<TPB> sh;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int r = blockIdx.x / a.splits, c = blockIdx.x - r * a.splits;
    if (a.finished && (a.finished[r] || a.scores[r] == -INFINITY)) return;
    const WordSource<T> src{a.rows.row(r), c * a.chunk, min(a.chunk, a.rows.V - c * a.chunk)};
    const int pieces = src.pieces(), full = src.n / T::vec;
    const char *base = src.row + (int64_t)src.first * T::bytes;

    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    float ref = -FLT_MAX, sum = 0.f;      // sum exp(z - ref) so far
    auto take = [&](const Raw &x, float &t) {
#pragma unroll
        for (int e = 0; e < T::vec; ++e) t = fmaxf(t, element<T>(x, e));
    };
    auto add = [&](const Raw &x) {
#pragma unroll
        for (int e = 0; e < T::vec; ++e) sum += __builtin_amdgcn_exp2f((fmaxf(element<T>(x, e), -INFINITY) - ref) * kLog2e);
    };
    auto rescale = [&]() {
        const float m = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), ref);
        if (m > ref) { sum *= __builtin_amdgcn_exp2f((ref - m) * kLog2e); ref = m; }
    };
    Raw held[HELD ? 4 : 1];
    if constexpr (HELD) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (tid + u * TPB < pieces) held[u] = src.load(tid + u * TPB);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (tid + u * TPB < pieces) take(held[u], top[u]);
        if constexpr (LSE) {
            rescale();
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (tid + u * TPB < pieces) add(held[u]);
        }
    } else {
        int p = tid;
        for (; p + 3 * TPB < full; p += 4 * TPB) {
            Raw x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = load16<T>(base + (int64_t)(p + u * TPB) * 16);
#pragma unroll
            for (int u = 0; u < 4; ++u) take(x[u], top[u]);
            if constexpr (LSE) {
                rescale();
#pragma unroll
                for (int u = 0; u < 4; ++u) add(x[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (p + u * TPB < pieces) {
                const Raw x = src.load(p + u * TPB);
                take(x, top[u]);
                if constexpr (LSE) { rescale(); add(x); }
            }
    }
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const uint32_t k = tid + u * TPB < pieces ? order_key(top[u]) : 0u;
        sh.keys[u * TPB + tid] = k;
        most = max(most, k);
    }
    sh.thread_keys[tid] = most;

    if constexpr (LSE) {
        const float m = wave_reduce(ref, [](float x, float y) { return fmaxf(x, y); });
        if (lane == 0) sh.ref[wave] = m;
        __syncthreads();
        float all = sh.ref[0];
        for (int w = 1; w < TPB / 64; ++w) all = fmaxf(all, sh.ref[w]);
        double s = (double)sum * (double)__builtin_amdgcn_exp2f((ref - all) * kLog2e);
        s = wave_reduce(s, [](double x, double y) { return x + y; });
        if (lane == 0) sh.sum[wave] = s;
        __syncthreads();
        if (tid == 0) {
            s = sh.sum[0];
            for (int w = 1; w < TPB / 64; ++w) s += sh.sum[w];
            if (a.parts) a.parts[blockIdx.x] = LsePart{s, all, 0.f};
            else a.lse[r] = all == INFINITY ? INFINITY : (float)((double)all + log(s));
        }
    }
    int n;
    if constexpr (HELD) {
        n = find_candidates<TPB>(src, sh, a.K, [&](uint32_t bound) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (sh.keys[u * TPB + tid] >= bound && tid + u * TPB < pieces) {
#pragma unroll
                    for (int e = 0; e < T::vec; ++e) {
                        const uint64_t x = src.entry(held[u], tid + u * TPB, e);
                        if (x && (uint32_t)(x >> 32) >= bound) {
                            const int at = atomicAdd(&sh.count, 1);
                            if (at < kCap) sh.cand[at] = x;
                        }
                    }
                }
        });
    } else {
        n = find_candidates<TPB>(src, sh, a.K, nullptr);
    }
    __syncthreads();
    if (a.keys) {
        uint64_t *out = a.keys + (int64_t)blockIdx.x * a.K;
        rank_candidates<TPB>(sh, n, a.K, [&](int place, uint64_t x) { out[place] = x; });
        for (int i = n + tid; i < a.K; i += TPB) out[i] = 0ull;
    } else {
        rank_candidates<TPB>(sh, n, a.K, [&](int place, uint64_t x) { put_out<T>(a, (int64_t)r * a.K + place, x); });
    }
}

// Joins the chunks of a row.
template <class T, int TPB>
__global__ __launch_bounds__(TPB) void top_join_kernel(TopArgs a) {
    __shared__ TopShared<TPB> sh;
    const int r = blockIdx.x, tid = threadIdx.x;
    const EntrySource src{a.keys + (int64_t)r * a.splits * a.K, a.splits * a.K};
    uint32_t top[4] = {0, 0, 0, 0};
    for (int p = tid; p < src.n; p += 4 * TPB) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (p + u * TPB < src.n) top[u] = max(top[u], (uint32_t)(src.list[p + u * TPB] >> 32));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) sh.keys[u * TPB + tid] = top[u];
    sh.thread_keys[tid] = max(max(top[0], top[1]), max(top[2], top[3]));
    if (a.lse && tid >= TPB - 64) {        // the last wave: the first one looks for the bound
        const double total = join_lse(a.parts + (int64_t)r * a.splits, a.splits);
        if (tid == TPB - 1) a.lse[r] = (float)total;
    }
    const int n = find_candidates<TPB>(src, sh, a.K, nullptr);
    __syncthreads();
    rank_candidates<TPB>(sh, n, a.K, [&](int place, uint64_t x) { put_out<T>(a, (int64_t)r * a.K + place, x); });
}

// Vocabularies of at most 64 words: L lanes per row, a word per lane, a word's place counted against the other lanes'.
template <class T, int L>
__global__ __launch_bounds__(256) void top_small_kernel(TopArgs a, int rows) {
    const int r = blockIdx.x * (256 / L) + threadIdx.x / L, v = threadIdx.x & (L - 1);
    const bool in = r < rows && v < a.rows.V;
    const float z = in ? load1<T>(a.rows.row(r), v) : -INFINITY;
    const uint64_t x = in ? pair_key(order_key(z), v) : 0ull;
    int place = 0;
#pragma unroll
    for (int j = 0; j < L; ++j) place += __shfl(x, j, L) > x ? 1 : 0;
    if (in && place < a.K) put_out<T>(a, (int64_t)r * a.K + place, x);
    if (a.lse) {
        float m = fmaxf(z, -FLT_MAX);
#pragma unroll
        for (int d = L / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, L));
        float s = __builtin_amdgcn_exp2f((fmaxf(z, -INFINITY) - m) * kLog2e);
#pragma unroll
        for (int d = L / 2; d; d >>= 1) s += __shfl_xor(s, d, L);
        if (r < rows && v == 0) a.lse[r] = m == INFINITY ? INFINITY : m + logf(s);
    }
}

// A wave per row where a wave's 256 groups suffice for K and a row is short: no barrier is waited at.
bool one_wave(const gscan_rows &rows, int K) { return K <= 64 && rows.V <= 2048; }

template <class T, int TPB>
int launch_rows(const TopArgs &a, int64_t grid, bool lse, hipStream_t stream) {
    const dim3 blocks((unsigned)grid);
    const bool held = a.chunk <= 4 * TPB * T::vec;
    if (lse && held) hipLaunchKernelGGL((top_row_kernel<T, TPB, true, true>), blocks, dim3(TPB), 0, stream, a);
    else if (lse) hipLaunchKernelGGL((top_row_kernel<T, TPB, true, false>), blocks, dim3(TPB), 0, stream, a);
    else if (held) hipLaunchKernelGGL((top_row_kernel<T, TPB, false, true>), blocks, dim3(TPB), 0, stream, a);
    else hipLaunchKernelGGL((top_row_kernel<T, TPB, false, false>), blocks, dim3(TPB), 0, stream, a);
    GSCAN_LAUNCHED("top_row_kernel");
    return 0;
}
template <class T>
int launch_rows(const TopArgs &a, int64_t grid, bool lse, bool wave, hipStream_t stream) {
    return wave ? launch_rows<T, 64>(a, grid, lse, stream) : launch_rows<T, 256>(a, grid, lse, stream);
}

template <class T>
int launch_small(const TopArgs &a, int rows, hipStream_t stream) {
    const int V = a.rows.V;
    if (V <= 8) hipLaunchKernelGGL((top_small_kernel<T, 8>), dim3(cdiv(rows, 32)), dim3(256), 0, stream, a, rows);
    else if (V <= 16) hipLaunchKernelGGL((top_small_kernel<T, 16>), dim3(cdiv(rows, 16)), dim3(256), 0, stream, a, rows);
    else if (V <= 32) hipLaunchKernelGGL((top_small_kernel<T, 32>), dim3(cdiv(rows, 8)), dim3(256), 0, stream, a, rows);
    else hipLaunchKernelGGL((top_small_kernel<T, 64>), dim3(cdiv(rows, 4)), dim3(256), 0, stream, a, rows);
    GSCAN_LAUNCHED("top_small_kernel");
    return 0;
}

template <class T>
int launch_join(const TopArgs &a, int rows, hipStream_t stream) {
    hipLaunchKernelGGL((top_join_kernel<T, 256>), dim3(rows), dim3(256), 0, stream, a);
    GSCAN_LAUNCHED("top_join_kernel");
    return 0;
}

#define BY_TYPE(type, call_f32, call_bf16, call_f16) \
    ((type) == GSCAN_F32 ? (call_f32) : (type) == GSCAN_BF16 ? (call_bf16) : (call_f16))
}  // namespace

int check_rows(const char *who, const gscan_rows *rows) {
    GSCAN_CHECK(rows, "%s: rows is NULL", who);
    GSCAN_CHECK(rows->data, "%s: logits are NULL", who);
    GSCAN_CHECK(rows->type == GSCAN_F32 || rows->type == GSCAN_BF16 || rows->type == GSCAN_F16, "%s: unknown type %d", who, rows->type);
    GSCAN_CHECK(rows->V >= 1 && rows->V <= (1 << 30), "%s: %d words (1 to 2^30)", who, rows->V);
    GSCAN_CHECK(rows->outer >= 1 && rows->inner >= 1 && rows->outer <= (1 << 24) && rows->inner <= (1 << 24) &&
                    rows->outer * rows->inner <= (1 << 24),
                "%s: %lld x %lld rows (1 to 2^24)", who, (long long)rows->outer, (long long)rows->inner);
    GSCAN_CHECK(rows->stride_outer >= 0 && rows->stride_inner >= 0, "%s: negative stride", who);
    const int64_t b = rows->type == GSCAN_F32 ? 4 : 2;
    GSCAN_CHECK(((uintptr_t)rows->data) % b == 0, "%s: logits are not aligned to their type", who);
    return 0;
}

TopChunks top_chunks(const gscan_rows &rows, int K) {
    const int64_t n = rows.outer * rows.inner;
    int splits = 1;
    // few rows: a row is split until there are about two workgroups per CU, chunks no shorter than 4096 words and 16 K
    const int least = std::max(4096, 16 * K);
    while (n * splits < 512 && rows.V / (2 * splits) >= least) splits *= 2;
    const int chunk = (cdiv(rows.V, splits) + 7) / 8 * 8;
    return TopChunks{cdiv(rows.V, chunk), chunk};
}

int top_chunk_keys(const gscan_rows &rows, int K, TopChunks c, uint64_t *keys, LsePart *parts, const uint8_t *finished,
                   const float *scores, hipStream_t stream) {
    TopArgs a{};
    a.rows = device_rows(rows);
    a.K = K; a.splits = c.splits; a.chunk = c.chunk;
    a.keys = keys; a.parts = parts; a.finished = finished; a.scores = scores;
    const int64_t grid = rows.outer * rows.inner * c.splits;
    const bool wave = one_wave(rows, K);
    return BY_TYPE(rows.type, launch_rows<TypeF32>(a, grid, parts != nullptr, wave, stream),
                   launch_rows<TypeBF16>(a, grid, parts != nullptr, wave, stream),
                   launch_rows<TypeF16>(a, grid, parts != nullptr, wave, stream));
}

size_t top_logits_workspace(const gscan_rows &rows, int K) {
    if (rows.V <= 64) return 0;
    const TopChunks c = top_chunks(rows, K);
    return c.splits == 1 ? 0 : (size_t)(rows.outer * rows.inner) * c.splits * (K * sizeof(uint64_t) + sizeof(LsePart));
}

int top_logits(const gscan_rows &rows, int K, void *values, int32_t *indices, float *lse, void *workspace, size_t bytes,
               hipStream_t stream) {
    GSCAN_CHECK(values && indices, "top_logits: NULL output");
    GSCAN_CHECK(K >= 1 && K <= kMaxTop && K <= rows.V, "top_logits: K = %d (1 to %d, at most the %d words of a row)", K, kMaxTop, rows.V);
    const int n = (int)(rows.outer * rows.inner);
    TopArgs a{};
    a.rows = device_rows(rows);
    a.K = K; a.values = values; a.indices = indices; a.lse = lse;
    if (rows.V <= 64)
        return BY_TYPE(rows.type, launch_small<TypeF32>(a, n, stream), launch_small<TypeBF16>(a, n, stream),
                       launch_small<TypeF16>(a, n, stream));
    const TopChunks c = top_chunks(rows, K);
    a.splits = c.splits; a.chunk = c.chunk;
    if (c.splits == 1)
        return BY_TYPE(rows.type, launch_rows<TypeF32>(a, n, lse != nullptr, one_wave(rows, K), stream),
                       launch_rows<TypeBF16>(a, n, lse != nullptr, one_wave(rows, K), stream),
                       launch_rows<TypeF16>(a, n, lse != nullptr, one_wave(rows, K), stream));
    const size_t need = top_logits_workspace(rows, K);
    GSCAN_CHECK(workspace && bytes >= need, "top_logits: workspace of %zu bytes, %zu needed", workspace ? bytes : (size_t)0, need);
    GSCAN_CHECK((uintptr_t)workspace % 8 == 0, "top_logits: workspace is not aligned to 8 bytes");
    a.parts = lse ? (LsePart *)workspace : nullptr;
    a.keys = (uint64_t *)((LsePart *)workspace + (size_t)n * c.splits);
    TRY_RC(top_chunk_keys(rows, K, c, a.keys, a.parts, nullptr, nullptr, stream));
    return BY_TYPE(rows.type, launch_join<TypeF32>(a, n, stream), launch_join<TypeBF16>(a, n, stream),
                   launch_join<TypeF16>(a, n, stream));
}

}  // namespace gscan
