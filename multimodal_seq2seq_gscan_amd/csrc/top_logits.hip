// The K best words of every row of logits, in order, with the row's log-sum-exp: what a teacher leaves for its student
// (distill.hip) and what a beam search looks at in a step (beam.hip).  Order: value descending, index ascending; a NaN counts
// as -inf.
//
// One pass over the row.  Every thread keeps the maximum of the words that it has seen (four maxima for a large K); at least K
// words are >= the K-th largest of these maxima, so it bounds the K-th largest word from below.  LDS holds 16 bits of the
// maximum of every 16-byte piece: the few pieces that reach the bound are read again, their words >= the bound (little more
// than K unless many are equal) are ranked by counting.  Without the pieces' maxima a thread's whole share of the row would be
// read again for every thread above the bound, a 128-byte line for every 16 bytes: 73 against 61 us for 4088 rows of 32000
// bfloat16 words, K = 64 (4.3 TB/s; a copy of 1 GiB reads and writes 5.05).  Few rows are split over workgroups and joined: one
// row of 131072 float words takes 8 + 7.5 us, latencies (a dozen dependent steps each) and no bytes.
// Exact for any input: where the words >= the bound do not fit the list, words above it and, in index order, words equal to
// it are taken apart, and if even the words above it do not fit (a row laid out against the threads), a radix selection over
// the row finds the K-th key.
#include <cstddef>

#include "logits.h"

namespace gscan {

namespace {
constexpr int kHits = 1024;        // groups of pieces that reach the bound
constexpr int kGroupList = 96;     // words of a short row that reach the bound

struct TopArgs {
    Rows rows;
    int K, splits, chunk;
    void *values; int32_t *indices; float *lse;      // splits == 1
    uint64_t *keys; LsePart *parts;                  // otherwise (and for the beam step)
    const uint8_t *finished; const float *scores;    // beam step: a row that is finished or has no score is left out
};

// What is looked for: entries whose key is > `key`, or >= it.
struct Limit {
    uint32_t key;
    bool equal;
    float value;          // of the key, and whether every word reaches it
    bool all;
    __device__ __forceinline__ Limit(uint32_t k, bool eq) : key(k), equal(eq), value(key_value(k)), all(eq && k <= 0x007fffffu) {}
};

// Words of a row (or of a part of it), 16 bytes at a time.
template <class T>
struct WordSource {
    static constexpr int vec = T::vec;
    typedef Raw Piece;
    const char *row;      // of the whole row
    int first, n;         // the part: words [first, first + n), first a multiple of vec
    __device__ __forceinline__ int pieces() const { return (n + vec - 1) / vec; }
    __device__ __forceinline__ Raw load(int p) const { return load_group<T>(row + (int64_t)first * T::bytes, p, n); }
    // (a NaN is below every limit but that of -inf)
    __device__ __forceinline__ bool reaches(const Raw &r, int p, int e, const Limit &l) const {
        const float z = element<T>(r, e);
        return (l.all || z > l.value || (l.equal && z == l.value)) && p * vec + e < n;
    }
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
    typedef uint64_t Piece;
    const uint64_t *list;
    int n;
    __device__ __forceinline__ int pieces() const { return n; }
    __device__ __forceinline__ uint64_t load(int p) const { return list[p]; }
    __device__ __forceinline__ bool reaches(uint64_t r, int, int, const Limit &l) const {
        const uint32_t k = pair_value(r);
        return k > l.key || (l.equal && k == l.key && k);
    }
    __device__ __forceinline__ uint64_t entry(uint64_t r, int, int) const { return r; }
    __device__ __forceinline__ uint64_t at(int i) const { return list[i]; }
};

// PIECES: how many pieces' (or groups of pieces') maxima are held, 0 for none.
template <int TPB, int PIECES>
struct TopShared {
    // candidates: at least 4 K (a wave takes K <= 64); pieces that reach the bound, where they need not be read again
    static constexpr int kCap = TPB == 64 ? 512 : 1024, kStash = TPB == 64 ? 256 : 512;
    union {
        alignas(16) uint64_t cand[kCap + 2];
        uint32_t keys[4 * TPB];         // four maxima a thread, until there is a bound; the radix selection's histogram
    };
    uint32_t thread_keys[TPB];
    alignas(16) uint16_t piece[PIECES ? PIECES : 1];
    alignas(16) Raw stash[PIECES ? 1 : kStash];
    uint16_t hit[PIECES ? kHits : kStash];
    uint32_t bound;
    int hits, count, above;
    int wave_count[TPB / 64];
    double sum[TPB / 64];
    float ref[TPB / 64];
};

// The thread's number with the waves turned round by the workgroup's: what few waves of a workgroup do falls on another of the
// CU's four SIMDs from one workgroup to the next.
template <int TPB>
__device__ __forceinline__ int turned() { return (int)((threadIdx.x + 64 * blockIdx.x) & (TPB - 1)); }

// Place for `total` entries (the same in every lane) behind a list's; one atomic a wave.
__device__ __forceinline__ int reserve(int *count, int total) {
    int at = 0;
    if ((threadIdx.x & 63) == 0) at = atomicAdd(count, total);
    return __builtin_amdgcn_readfirstlane(at);
}
__device__ __forceinline__ int lanes_before(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}
// Puts the entries of a piece a lane that reach the limit on the list of candidates; every lane of a wave takes part, one
// without a piece with p behind the last.  What does not fit is counted only.
template <class S, class Sh>
__device__ __forceinline__ void push_piece(const S &src, Sh &sh, const typename S::Piece &raw, int p, const Limit &l) {
    unsigned long long b[S::vec];
    int total = 0;
#pragma unroll
    for (int e = 0; e < S::vec; ++e) {
        b[e] = __ballot(p < src.pieces() && src.reaches(raw, p, e, l));
        total += __popcll(b[e]);
    }
    if (total == 0) return;
    int at = reserve(&sh.count, total);
#pragma unroll
    for (int e = 0; e < S::vec; ++e) {
        if (b[e] == 0) continue;
        const int mine = at + lanes_before(b[e]);
        if ((b[e] >> (threadIdx.x & 63) & 1) && mine < Sh::kCap) sh.cand[mine] = src.entry(raw, p, e);
        at += __popcll(b[e]);
    }
}
template <int TPB, class S, class Sh>
__device__ __forceinline__ void scan_all(const S &src, Sh &sh, uint32_t bound, bool equal) {
    const Limit l(bound, equal);
    for (int base = 0; base < src.pieces(); base += TPB) {
        const int p = base + (int)threadIdx.x;
        push_piece(src, sh, src.load(min(p, src.pieces() - 1)), p, l);
    }
}

// The first `want` entries, in index order, whose key is `key`, behind the `at` candidates that are there.
template <int TPB, class S, class Sh>
__device__ void collect_equal(const S &src, Sh &sh, uint32_t key, int at, int want) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int found = 0;
    for (int base = 0; base < src.n && found < want; base += TPB) {
        const int i = base + tid;
        const uint64_t x = i < src.n ? src.at(i) : 0ull;
        const bool is = x && pair_value(x) == key;
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
template <int TPB, class S, class Sh>
__device__ int radix_select(const S &src, Sh &sh, int K, uint32_t *key) {
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
                const uint32_t k = pair_value(src.entry(raw, p, e));
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

// With the threads' maxima in sh.thread_keys (and four a thread in sh.keys): leaves candidates that hold the K best entries in
// sh.cand and returns their number.  `scan(bound)` puts the entries >= bound on the list; it may leave some out where it
// counts more than fit.
template <int TPB, class S, class Sh, class F>
__device__ int find_candidates(const S &src, Sh &sh, int K, F scan) {
    const int tid = turned<TPB>();
    __syncthreads();
    if (tid < 64) {
        // K of TPB maxima bound nearly as well as K of four times as many, for a quarter of the counting, while K is no more
        // than a quarter of them
        const uint32_t b = 4 * K <= TPB ? kth_bound<TPB / 64>([&](int i) { return sh.thread_keys[i]; }, TPB, K, tid)
                                        : kth_bound<4 * TPB / 64>([&](int i) { return sh.keys[i]; }, 4 * TPB, K, tid);
        if (tid == 0) { sh.bound = b; sh.hits = 0; sh.count = 0; }
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    scan(bound);
    __syncthreads();
    int n = sh.count;
    if (n <= Sh::kCap) return n;
    auto again = [&](uint32_t key) {
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
        scan_all<TPB>(src, sh, key, false);
        __syncthreads();
        return sh.count;
    };
    n = again(bound);
    if (n >= K && n <= Sh::kCap) return n;
    if (n < K) {
        collect_equal<TPB>(src, sh, bound, n, K - n);
        return K;
    }
    __syncthreads();
    uint32_t key;
    const int equal = radix_select<TPB>(src, sh, K, &key);
    n = again(key);
    collect_equal<TPB>(src, sh, key, n, equal);
    return K;
}

// Every candidate's place is the number of candidates before it; `put(place, entry)` for the first K of them.
template <int TPB, class Sh, class F>
__device__ __forceinline__ void rank_candidates(Sh &sh, int n, int K, F put) {
    const int even = (n + 1) & ~1;
    __syncthreads();
    if (threadIdx.x == 0 && even > n) sh.cand[n] = 0;
    __syncthreads();
    for (int i = turned<TPB>(); i < n; i += TPB) {
        const uint64_t x = sh.cand[i];
        const double mine = pair_double(x);
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < even; j += 2) {
            const double2 q = *(const double2 *)&sh.cand[j];
            place += (q.x > mine ? 1 : 0) + (q.y > mine ? 1 : 0);
        }
        if (place < K) put(place, x);
    }
}

// A thread's sum exp(z - ref) over the words so far.  Near 0 as 2^(z log2 e + back), back = -ref log2 e rounded: one
// multiply-add a word; the sum is off by the factor 2^delta, delta = what the rounding added, which is known and is taken off
// when the reference changes and at the end (candidates of different beams are compared through this sum: 32 bits of it are
// not given away).  Far out, where delta grows, the distance from the reference comes first.
struct RunningSum {
    float sum = 0.f, ref = -FLT_MAX, back = 0.f, delta = 0.f;
    bool near = false;
    __device__ __forceinline__ void clear() { sum = 0.f; }
    __device__ __forceinline__ void grow(float m) {
        if (m > ref) {
            const bool n = fabsf(m) < 65536.f;
            const float b = n ? -m * kLog2e : 0.f, d = n ? fmaf(m, kLog2e, b) : 0.f;
            sum *= __builtin_amdgcn_exp2f((ref - m) * kLog2e + (d - delta));
            ref = m; back = b; delta = d; near = n;
        }
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&z)[N]) {
        if (near) {
#pragma unroll
            for (int e = 0; e < N; ++e) sum += __builtin_amdgcn_exp2f(fmaf(z[e], kLog2e, back));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) sum += __builtin_amdgcn_exp2f((z[e] - ref) * kLog2e);
        }
    }
    __device__ __forceinline__ void add_word(float z) {
        const float one[1] = {z};
        add(one);
    }
    __device__ __forceinline__ double relative_to(float m) const {
        // 2^-delta to the first order: delta is below 2^-7
        const double d = (double)delta * 0.6931471805599453;
        return (double)sum * (1.0 - d + 0.5 * d * d) * (double)__builtin_amdgcn_exp2f((ref - m) * kLog2e);
    }
};

template <class T>
__device__ __forceinline__ void put_out(const TopArgs &a, int64_t at, uint64_t x) {
    store1<T>((char *)a.values, at, key_value(pair_value(x)));
    a.indices[at] = pair_index(x);
}

// The maxima of a piece's quarters, as ordered numbers; 0 without a piece.  (Words behind the row's end are -inf: a bound that
// they take part in is -inf, which every word reaches.)
template <class T>
__device__ __forceinline__ void quarters(const Raw &x, bool there, uint32_t (&q)[4]) {
    constexpr int Q = T::vec / 4;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        float t = element<T>(x, u * Q);
#pragma unroll
        for (int e = 1; e < Q; ++e) t = fmaxf(t, element<T>(x, u * Q + e));
        q[u] = there ? order_key(t) : 0u;
    }
}

// One workgroup per row, or per chunk of a row.  PIECES = 0: at most four pieces a thread, which stay in registers: nothing is
// read again.
template <class T, int TPB, bool LSE, int PIECES>
__global__ __launch_bounds__(TPB) void top_row_kernel(TopArgs a) {
    __shared__ TopShared<TPB, PIECES> sh;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int r = blockIdx.x / a.splits, c = blockIdx.x - r * a.splits;
    if (a.finished && (a.finished[r] || a.scores[r] == -INFINITY)) return;
    const WordSource<T> src{a.rows.row(r), c * a.chunk, min(a.chunk, a.rows.V - c * a.chunk)};
    const int pieces = src.pieces(), full = src.n / T::vec;
    const char *base = src.row + (int64_t)src.first * T::bytes;

    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    RunningSum sum;
    auto largest = [&](const Raw &x) {
        float t = element<T>(x, 0);
#pragma unroll
        for (int e = 1; e < T::vec; ++e) t = fmaxf(t, element<T>(x, e));
        return fmaxf(t, -INFINITY);
    };
    auto rescale = [&]() { sum.grow(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))); };
    auto add = [&](const Raw &x) {
        float z[T::vec];
#pragma unroll
        for (int e = 0; e < T::vec; ++e) z[e] = element<T>(x, e);
        sum.add(z);
    };
    Raw held[PIECES ? 1 : 4];
    // group (s, t) of pieces: t + TPB (per s + k), k < per
    const int steps = (pieces + TPB - 1) / TPB, per = PIECES ? max(1, (steps + PIECES / TPB - 1) / (PIECES / TPB)) : 1;
    if constexpr (PIECES == 0) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (tid + u * TPB < pieces) held[u] = src.load(tid + u * TPB);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (tid + u * TPB < pieces) top[u] = largest(held[u]);
        if constexpr (LSE) {
            rescale();
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (tid + u * TPB < pieces) add(held[u]);
        }
    } else {
        float group = -INFINITY;
        int s = 0, k = 0;
        auto take = [&](const Raw &x, float &t) {
            const float m = largest(x);
            t = fmaxf(t, m);
            group = fmaxf(group, m);
            if (++k == per) {
                sh.piece[s * TPB + tid] = (uint16_t)(order_key(group) >> 16);
                group = -INFINITY; k = 0; ++s;
            }
        };
        int p = tid;
        for (; p + 3 * TPB < full; p += 4 * TPB) {
            Raw x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = load16<T, true>(base + (int64_t)(p + u * TPB) * 16);
#pragma unroll
            for (int u = 0; u < 4; ++u) take(x[u], top[u]);
            if constexpr (LSE) {
                rescale();
                float z[4 * T::vec];
#pragma unroll
                for (int i = 0; i < 4 * T::vec; ++i) z[i] = element<T>(x[i / T::vec], i % T::vec);
                sum.add(z);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (p + u * TPB < pieces) {
                const Raw x = src.load(p + u * TPB);
                take(x, top[u]);
                if constexpr (LSE) { rescale(); add(x); }
            }
        // a group that is not full, and those that this thread has no piece of
        const int groups = (steps + per - 1) / per;
        if (k) { sh.piece[s * TPB + tid] = (uint16_t)(order_key(group) >> 16); ++s; }
        for (; s < groups; ++s) sh.piece[s * TPB + tid] = 0;
    }
    uint32_t most = 0, four[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        four[u] = tid + u * TPB < pieces ? order_key(top[u]) : 0u;
        most = max(most, four[u]);
    }
    sh.thread_keys[tid] = most;
    if (4 * a.K > TPB) {
        if constexpr (PIECES == 0) {
            // one or two pieces a thread: maxima of quarters or halves of them, or a large K is bounded by hardly more than
            // the least of the maxima, and most words reach that (2000 bfloat16 words, K = 200: 777 for 135 us, 16384 rows)
            if (pieces <= TPB) {
                quarters<T>(held[0], tid < pieces, four);
            } else if (pieces <= 2 * TPB) {
                uint32_t q[4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    quarters<T>(held[u], tid + u * TPB < pieces, q);
                    four[2 * u] = max(q[0], q[1]);
                    four[2 * u + 1] = max(q[2], q[3]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) sh.keys[u * TPB + tid] = four[u];
    }

    if constexpr (LSE) {
        if (sum.sum != sum.sum) {          // a NaN among the words (or an infinity): they count as -inf
            sum.clear();
            for (int p = tid; p < pieces; p += TPB) {
                const Raw x = src.load(p);
#pragma unroll
                for (int e = 0; e < T::vec; ++e) sum.add_word(fmaxf(element<T>(x, e), -INFINITY));
            }
        }
        const float m = wave_max(sum.ref);
        if (lane == 0) sh.ref[wave] = m;
        __syncthreads();
        float all = sh.ref[0];
        for (int w = 1; w < TPB / 64; ++w) all = fmaxf(all, sh.ref[w]);
        double s = sum.relative_to(all);
        s = wave_reduce(s, [](double x, double y) { return x + y; });
        if (lane == 0) sh.sum[wave] = s;
        __syncthreads();
        if (tid == TPB - 1) {
            s = sh.sum[0];
            for (int w = 1; w < TPB / 64; ++w) s += sh.sum[w];
            if (a.parts) a.parts[blockIdx.x] = LsePart{s, all, 0.f};
            else a.lse[r] = all == INFINITY ? INFINITY : (float)((double)all + log(s));
        }
    }
    const int n = find_candidates<TPB>(src, sh, a.K, [&](uint32_t bound) {
        const Limit l(bound, true);
        if constexpr (PIECES == 0) {
            // a lane in sixteen holds such a piece: they are dealt out to a lane each before their words are looked at
            unsigned long long m[4];
            int total = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                m[u] = __ballot(tid + u * TPB < pieces && (l.all || top[u] >= l.value));
                total += __popcll(m[u]);
            }
            if (total) {
                int at = reserve(&sh.hits, total);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int mine = at + lanes_before(m[u]);
                    if ((m[u] >> lane & 1) && mine < sh.kStash) { sh.stash[mine] = held[u]; sh.hit[mine] = (uint16_t)(tid + u * TPB); }
                    at += __popcll(m[u]);
                }
            }
            __syncthreads();
            const int hits = sh.hits;
            if (hits > sh.kStash) {                   // (nearly) all words alike: the caller goes over the row
                if (tid == 0) sh.count = sh.kCap + 1;
                return;
            }
            for (int it = turned<TPB>(); (it & ~63) < hits; it += TPB) {
                const int at = min(it, sh.kStash - 1);
                push_piece(src, sh, sh.stash[at], it < hits ? (int)sh.hit[at] : pieces, l);
            }
        } else {
            const int groups = (steps + per - 1) / per * TPB;
            const uint32_t least = max(bound >> 16, 1u);
            constexpr int pairs = PIECES / TPB / 2;      // two groups' maxima at a time
            uint32_t two[pairs];
            int total = 0;
#pragma unroll
            for (int i = 0; i < pairs; ++i) {
                const int g = 2 * (tid + i * TPB);
                two[i] = g < groups ? *(const uint32_t *)&sh.piece[g] : 0u;
                total += __popcll(__ballot((two[i] & 0xffffu) >= least)) + __popcll(__ballot((two[i] >> 16) >= least));
            }
            if (total) {
                int at = reserve(&sh.hits, total);
#pragma unroll
                for (int i = 0; i < pairs; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool hit = (h ? two[i] >> 16 : two[i] & 0xffffu) >= least;
                        const unsigned long long m = __ballot(hit);
                        if (m == 0) continue;
                        const int mine = at + lanes_before(m);
                        if (hit && mine < kHits) sh.hit[mine] = (uint16_t)(2 * (tid + i * TPB) + h);
                        at += __popcll(m);
                    }
            }
            __syncthreads();
            const int hits = sh.hits, items = hits * per;
            if (hits > kHits) {                    // (nearly) all words alike: the caller goes over the row
                if (tid == 0) sh.count = sh.kCap + 1;
                return;
            }
            for (int it = turned<TPB>(); (it & ~63) < items; it += TPB) {
                int p = pieces;
                if (it < items) {
                    const int h = it / per, g = sh.hit[h];
                    p = (g & (TPB - 1)) + TPB * (per * (g / TPB) + it - h * per);
                }
                push_piece(src, sh, src.load(min(p, pieces - 1)), p, l);
            }
        }
    });
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
    __shared__ TopShared<TPB, 0> sh;
    const int r = blockIdx.x, tid = threadIdx.x;
    const EntrySource src{a.keys + (int64_t)r * a.splits * a.K, a.splits * a.K};
    uint32_t top[4] = {0, 0, 0, 0};
    for (int p = tid; p < src.n; p += 4 * TPB) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (p + u * TPB < src.n) top[u] = max(top[u], pair_value(src.list[p + u * TPB]));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) sh.keys[u * TPB + tid] = top[u];
    sh.thread_keys[tid] = max(max(top[0], top[1]), max(top[2], top[3]));
    if (a.lse && tid >= TPB - 64) {        // one wave (in three workgroups of four another one than looks for the bound)
        const double total = join_lse(a.parts + (int64_t)r * a.splits, a.splits);
        if (tid == TPB - 1) a.lse[r] = (float)total;
    }
    const int n = find_candidates<TPB>(src, sh, a.K, [&](uint32_t bound) { scan_all<TPB>(src, sh, bound, true); });
    rank_candidates<TPB>(sh, n, a.K, [&](int place, uint64_t x) { put_out<T>(a, (int64_t)r * a.K + place, x); });
}

// Short rows, few words looked for: sixteen lanes per row, P pieces a lane, held as numbers (a NaN behind the row's end, where
// no comparison is true).  A bound that K words reach comes from bisection, counting the pieces' maxima, or the words where a
// row has few pieces; the words that reach it go to a list in LDS and are ranked by counting.  Where more reach it than the
// list takes (many words alike), the K best are taken out one by one.  A row stays within its lanes: nothing waits at a barrier.
template <class T, int P, bool LSE>
__global__ __launch_bounds__(256) void top_group_kernel(TopArgs a, int rows) {
    constexpr int R = 16, N = T::vec, W = P * N;
    __shared__ alignas(16) uint64_t s_list[R][kGroupList + 2];
    const int slot = threadIdx.x >> 4, lane = threadIdx.x & 15, r = blockIdx.x * R + slot, V = a.rows.V, K = a.K;
    const bool live = r < rows && !(a.finished && (a.finished[r] || a.scores[r] == -INFINITY));
    const char *row = a.rows.row(r < rows ? r : 0);
    const int full = V / N, rest = V - full * N, pieces = full + (rest ? 1 : 0);
    uint64_t *list = s_list[slot];
    float z[W], most[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int p = lane + i * 16;
        Raw x{{0, 0, 0, 0}};
        if (live && p < full) x = load16<T, true>(row + (int64_t)p * 16);
        else if (live && p == full && rest) x = load_tail<T>(row, p * N, V);
        const int words = !live ? 0 : p < full ? N : p == full ? rest : 0;
#pragma unroll
        for (int e = 0; e < N; ++e) z[i * N + e] = e < words ? fmaxf(element<T>(x, e), -INFINITY) : NAN;
    }
    float lowest = NAN, zmax = NAN;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        most[i] = z[i * N];
#pragma unroll
        for (int e = 1; e < N; ++e) most[i] = fmaxf(most[i], z[i * N + e]);
        lowest = fminf(lowest, most[i]);
        zmax = fmaxf(zmax, most[i]);
    }
    lowest = group_reduce<16>(lowest, [](float u, float v) { return fminf(u, v); });
    zmax = group_reduce<16>(zmax, [](float u, float v) { return fmaxf(u, v); });
    auto plus = [](int u, int v) { return u + v; };
    auto index_of = [&](int i) { return (lane + i / N * 16) * N + i % N; };

    // count(>= lo) >= K and count(>= top) < K, of what is counted
    const bool by_piece = pieces >= 2 * K;
    uint32_t lo = pieces >= K ? order_key(lowest) : 0x007fffffu, top = order_key(zmax) + 1;
    bool found = !live || top - lo <= 1;
    while (__ballot(!found)) {
        const uint32_t mid = lo + (top - lo) / 2;
        const float v = key_value(mid);
        int c = 0;
        if (by_piece) {
#pragma unroll
            for (int i = 0; i < P; ++i) c += most[i] >= v ? 1 : 0;
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) c += z[i] >= v ? 1 : 0;
        }
        c = group_reduce<16>(c, plus);
        if (!found) {
            if (c >= K) { lo = mid; found = c <= K + (K >> 2); }
            else top = mid;
            found = found || top - lo <= 1;
        }
    }
    const float bound = key_value(lo);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) mine += z[i] >= bound ? 1 : 0;
    const int n = group_reduce<16>(mine, plus);
    int at = sum_before16(mine);
    const bool fits = n <= kGroupList;
    auto put = [&](int place, uint64_t x) {
        if (a.keys) a.keys[(int64_t)r * K + place] = x;
        else put_out<T>(a, (int64_t)r * K + place, x);
    };
    if (fits) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (z[i] >= bound) list[at++] = (uint64_t)__float_as_uint(z[i]) << 32 | (uint32_t)index_of(i);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = lane; i < n; i += 16) {
            const uint64_t x = list[i];
            list[i] = pair_key(order_key(__uint_as_float((uint32_t)(x >> 32))), (int)(uint32_t)x);
        }
        if (lane == 0) list[n] = 0;                        // a pair is compared at a time
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = lane; i < n; i += 16) {
            const uint64_t x = list[i];
            const double me = pair_double(x);
            int place = 0;
            for (int j = 0; j < n; j += 2) {
                const double2 q = *(const double2 *)&list[j];
                place += (q.x > me ? 1 : 0) + (q.y > me ? 1 : 0);
            }
            if (place < K) put(place, x);
        }
    }
    if constexpr (LSE) {
        const float m = fmaxf(zmax, -FLT_MAX);
        double sum = 0.0;                                  // of a piece in 32 bits, from there on in 64
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float s = 0.f;
#pragma unroll
            for (int e = i * N; e < i * N + N; ++e) s += z[e] == z[e] ? __builtin_amdgcn_exp2f((z[e] - m) * kLog2e) : 0.f;
            sum += s;
        }
        sum = group_reduce<16>(sum, [](double u, double v) { return u + v; });
        if (live && lane == 0) {
            if (a.parts) a.parts[r] = LsePart{sum, m, 0.f};
            else a.lse[r] = m == INFINITY ? INFINITY : (float)((double)m + log(sum));
        }
    }
    if (__ballot(!fits)) {
        for (int place = 0; place < K; ++place) {
            float best = NAN;
            int which = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (z[i] > best || (best != best && z[i] == z[i])) { best = z[i]; which = index_of(i); }
            const float all = group_reduce<16>(best, [](float u, float v) { return fmaxf(u, v); });
            const int first = group_reduce<16>(best == all ? which : 0x7fffffff, [](int u, int v) { return min(u, v); });
            if (!fits && first == which && best == all) {
                put(place, pair_key(order_key(best), first));
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (index_of(i) == first) z[i] = NAN;
            }
        }
    }
}

// Vocabularies of at most 16 words: L lanes per row, a word per lane, a word's place counted against the other lanes'.
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

// Short rows share a wave.  262144 rows against a wave per row (a word per lane up to 64 words): 20 words of float, K = 4: 42 for
// 86 us, 64 words: 46 for 335; 131072 rows, K = 4 / 32: 100 words of float 31 / 56 for 132 / 217, 200: 41 / 73 for 135 / 180, of
// bfloat16 500: 58 / 104 for 162 / 213; 65536 rows of 1000: 57 / 90 for 74 / 97.  Issue binds them: 262144 rows of 100
// words, K = 4, take 607 VALU instructions a wave of 4 rows, 1.04 per SIMD and four cycles (some take fewer), 131072 rows, K = 32:
// 1049 and 0.89.  9 words are faster a word per lane (25 for 43).
bool top_grouped(const gscan_rows &rows, int K) {
    return K <= 64 && rows.V > 16 && cdiv(rows.V, rows.type == GSCAN_F32 ? 4 : 8) <= 16 * 8;
}

// A wave per row where a wave's 256 groups suffice for K and a row is short: no barrier is waited at.
bool one_wave(const gscan_rows &rows, int K) { return K <= 64 && rows.V <= 2048; }

template <class T, int TPB, int PIECES>
int launch_rows(const TopArgs &a, int64_t grid, bool lse, hipStream_t stream) {
    const dim3 blocks((unsigned)grid);
    if (lse) hipLaunchKernelGGL((top_row_kernel<T, TPB, true, PIECES>), blocks, dim3(TPB), 0, stream, a);
    else hipLaunchKernelGGL((top_row_kernel<T, TPB, false, PIECES>), blocks, dim3(TPB), 0, stream, a);
    GSCAN_LAUNCHED("top_row_kernel");
    return 0;
}
// the pieces' maxima: all of them in 8 KB (rows of 32768 16-bit words), else in 16 KB, with groups of pieces from there on
template <class T, int TPB>
int launch_rows(const TopArgs &a, int64_t grid, bool lse, hipStream_t stream) {
    const int pieces = cdiv(a.chunk, T::vec);
    if (pieces <= 4 * TPB) return launch_rows<T, TPB, 0>(a, grid, lse, stream);
    if constexpr (TPB == 256 || T::vec == 4) {       // a wave's 2048 words at most: of 16 bits they are 4 pieces a lane
        if (TPB == 64 || pieces <= 16 * TPB) return launch_rows<T, TPB, 16 * TPB>(a, grid, lse, stream);
    }
    return launch_rows<T, 256, 32 * 256>(a, grid, lse, stream);
}
template <class T>
int launch_rows(const TopArgs &a, int64_t grid, bool lse, bool wave, hipStream_t stream) {
    return wave ? launch_rows<T, 64>(a, grid, lse, stream) : launch_rows<T, 256>(a, grid, lse, stream);
}

template <class T>
int launch_small(const TopArgs &a, int rows, hipStream_t stream) {
    const int V = a.rows.V;
    if (V <= 8) hipLaunchKernelGGL((top_small_kernel<T, 8>), dim3(cdiv(rows, 32)), dim3(256), 0, stream, a, rows);
    else hipLaunchKernelGGL((top_small_kernel<T, 16>), dim3(cdiv(rows, 16)), dim3(256), 0, stream, a, rows);
    GSCAN_LAUNCHED("top_small_kernel");
    return 0;
}

template <class T, int P>
int launch_group(const TopArgs &a, int rows, bool lse, hipStream_t stream) {
    const dim3 grid(cdiv(rows, 16));
    if (lse) hipLaunchKernelGGL((top_group_kernel<T, P, true>), grid, dim3(256), 0, stream, a, rows);
    else hipLaunchKernelGGL((top_group_kernel<T, P, false>), grid, dim3(256), 0, stream, a, rows);
    GSCAN_LAUNCHED("top_group_kernel");
    return 0;
}
template <class T>
int launch_group(const TopArgs &a, int rows, bool lse, hipStream_t stream) {
    const int pieces = cdiv(a.rows.V, T::vec);
    if (pieces <= 16) return launch_group<T, 1>(a, rows, lse, stream);
    if (pieces <= 32) return launch_group<T, 2>(a, rows, lse, stream);
    if (pieces <= 64) return launch_group<T, 4>(a, rows, lse, stream);
    return launch_group<T, 8>(a, rows, lse, stream);
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
    // a launch counts its threads in 32 bits: 512 a row
    GSCAN_CHECK(rows->outer >= 1 && rows->inner >= 1 && rows->outer < (1 << 23) && rows->inner < (1 << 23) &&
                    rows->outer * rows->inner < (1 << 23),
                "%s: %lld x %lld rows (1 to 2^23 - 1)", who, (long long)rows->outer, (long long)rows->inner);
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
    if (top_grouped(rows, K))
        return BY_TYPE(rows.type, launch_group<TypeF32>(a, (int)grid, parts != nullptr, stream),
                       launch_group<TypeBF16>(a, (int)grid, parts != nullptr, stream),
                       launch_group<TypeF16>(a, (int)grid, parts != nullptr, stream));
    const bool wave = one_wave(rows, K);
    return BY_TYPE(rows.type, launch_rows<TypeF32>(a, grid, parts != nullptr, wave, stream),
                   launch_rows<TypeBF16>(a, grid, parts != nullptr, wave, stream),
                   launch_rows<TypeF16>(a, grid, parts != nullptr, wave, stream));
}

size_t top_logits_workspace(const gscan_rows &rows, int K) {
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
    if (top_grouped(rows, K))
        return BY_TYPE(rows.type, launch_group<TypeF32>(a, n, lse != nullptr, stream), launch_group<TypeBF16>(a, n, lse != nullptr, stream),
                       launch_group<TypeF16>(a, n, lse != nullptr, stream));
    if (rows.V <= 16)
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
