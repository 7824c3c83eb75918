// One step of beam search: the W best continuations of a batch row's W beams, and the beams' states put in the new order.
//
// A candidate (w, v) has the score  score_w + z[w, v] - lse(z[w, :]);  a finished beam has one candidate, itself with its
// score as it is and a padding word.  The order is score descending, then w ascending, then, within a beam, logit descending (which
// decides where scores that lie far out round to the same number) and v ascending.  Within a beam that is the order of the
// logits alone, so the W best of every beam (top_logits.hip, one pass over the logits, with the beam's softmax sum) hold the W best
// of all: W sorted lists (W times the chunks of a row) that one wave merges by W rounds over the lists' heads.  Scores are
// compared in 64 bits: candidates of different beams come closer to each other than 32 bits of a sum tell apart.  A beam whose
// candidates all score -inf whatever their logits (its own score is -inf or NaN, or its logits have no log-softmax) has them in
// the order of v.
#include "logits.h"

namespace gscan {

namespace {
struct BeamArgs {
    Rows rows;
    int B, W, K, splits, eos, pad;
    const float *scores; const uint8_t *finished;
    const uint64_t *keys; const LsePart *parts;
    float *scores_out; int32_t *parents; int64_t *tokens; uint8_t *finished_out;
};
constexpr int kMaxEntries = 4096;        // list entries of a batch row held in LDS

__device__ __forceinline__ double score_value(uint64_t key) {
    return __longlong_as_double((int64_t)(key ^ ((key >> 63) ? 0x8000000000000000ull : ~0ull)));
}

__device__ __forceinline__ void put_beam(const BeamArgs &a, int b, int place, uint64_t key, uint32_t flat) {
    const int w = (int)(flat / (uint32_t)a.rows.V), v = (int)(flat - (uint32_t)w * (uint32_t)a.rows.V);
    const int64_t at = (int64_t)b * a.W + place;
    a.scores_out[at] = (float)score_value(key);
    a.parents[at] = w;
    a.tokens[at] = v;
    a.finished_out[at] = a.finished[(int64_t)b * a.W + w] || v == a.eos ? 1 : 0;
}

// score_w + z - lse as an ordered number; what is not a number counts as -inf
__device__ __forceinline__ uint64_t score_key(double score, double z, double lse) {
    const double s = score + (z - lse);
    return order_key64(s == s ? s : -INFINITY);
}

// whether the logits of a beam order its candidates (else all of them score -inf)
__device__ __forceinline__ bool by_logit(float score, double lse) { return score > -INFINITY && fabs(lse) < INFINITY; }

// Joins the lists of a batch row's beams: W rounds of one wave, each a reduction and one lane's two LDS reads, behind the lists'
// way into LDS.  Latencies bind it: 5.8 us for one row's 16 lists of 4, 10.5 for 32 rows' 16 lists of 8.
__global__ __launch_bounds__(256) void beam_join_kernel(BeamArgs a) {
    extern __shared__ uint64_t s_key[];          // [entries], then uint32 flat[entries], then int head[lists]
    __shared__ double s_lse[kMaxBeams];
    __shared__ float s_score[kMaxBeams];
    __shared__ uint8_t s_done[kMaxBeams];
    const int b = blockIdx.x, tid = threadIdx.x, lists = a.W * a.splits, n = lists * a.K;
    uint32_t *s_flat = (uint32_t *)(s_key + n);
    int *s_head = (int *)(s_flat + n);
    const int64_t row0 = (int64_t)b * a.W;
    const uint64_t *keys = a.keys + row0 * a.splits * a.K;
    // what a beam that is finished or has no score has left there is not looked at
    const uint64_t early = tid < n ? keys[tid] : 0ull;
    if (tid < a.W) { s_score[tid] = a.scores[row0 + tid]; s_done[tid] = a.finished[row0 + tid]; }
    for (int w = tid >> 6; w < a.W; w += 4) {
        const double lse = join_lse(a.parts + (row0 + w) * a.splits, a.splits);
        if ((tid & 63) == 0) s_lse[w] = lse;
    }
    for (int l = tid; l < lists; l += 256) s_head[l] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += 256) {
        const int l = i / a.K, k = i - l * a.K, w = l / a.splits, c = l - w * a.splits;
        const float score = s_score[w];
        uint64_t key = 0;
        uint32_t v = 0;
        if (s_done[w]) {
            if (c == 0 && k == 0) { key = score_key((double)score, 0.0, 0.0); v = (uint32_t)a.pad; }
        } else if (!by_logit(score, s_lse[w])) {
            if (c == 0) { key = order_key64(-INFINITY); v = (uint32_t)k; }
        } else {
            const uint64_t x = i == tid ? early : keys[i];
            if (x) { key = score_key((double)score, (double)key_value(pair_value(x)), s_lse[w]); v = (uint32_t)pair_index(x); }
        }
        s_key[i] = key;
        s_flat[i] = (uint32_t)w * (uint32_t)a.rows.V + v;
    }
    __syncthreads();
    if (tid >= 64) return;
    // lane l owns the lists l, l + 64, ...: its best head, then the best of all lanes', W times
    uint64_t best = 0;
    uint32_t flat = ~0u;
    int from = -1;
    // what decides between the heads of two lists of one beam whose scores are equal: the larger comes first
    auto within = [&](int l, int w) {
        const int i = l * a.K + s_head[l];
        return s_done[w] || !by_logit(s_score[w], s_lse[w]) ? pair_key(0u, (int)(s_flat[i] - (uint32_t)w * (uint32_t)a.rows.V)) : keys[i];
    };
    auto before = [&](int l, int m) {
        const int w = l / a.splits, o = m / a.splits;
        return w != o ? w < o : within(l, w) > within(m, o);
    };
    auto refresh = [&]() {
        best = 0; flat = ~0u; from = -1;
        for (int l = tid; l < lists; l += 64) {
            const int h = s_head[l];
            if (h >= a.K) continue;
            const uint64_t k = s_key[l * a.K + h];
            if (k > best || (k == best && k && before(l, from))) { best = k; flat = s_flat[l * a.K + h]; from = l; }
        }
    };
    auto largest = [](uint32_t x, uint32_t y) { return max(x, y); };
    refresh();
    for (int place = 0; place < a.W; ++place) {
        // the high words settle it unless two scores come within 2^-20 of each other
        uint32_t high = wave_reduce((uint32_t)(best >> 32), largest);
        bool in = (uint32_t)(best >> 32) == high;
        if (__popcll(__ballot(in)) > 1) {
            const uint32_t low = wave_reduce(in ? (uint32_t)best : 0u, largest);
            in = in && (uint32_t)best == low && from >= 0;
            if (__popcll(__ballot(in)) > 1) {        // equal: the lowest beam, then (chunks of one row) as `within` says
                const int w = in ? from / a.splits : kMaxBeams, lowest = wave_reduce(w, [](int x, int y) { return min(x, y); });
                in = in && w == lowest;
                const double x = in ? pair_double(within(from, w)) : -1.0, first = wave_reduce(x, [](double u, double v) { return fmax(u, v); });
                in = in && x == first;
            }
        }
        if (in && from >= 0) {                       // one lane: heads of one beam differ in their words
            s_head[from] += 1;
            put_beam(a, b, place, best, flat);
            refresh();
        }
    }
}

// Vocabularies of at most 64 words: L lanes per beam, a word per lane, a candidate's place counted against all of its batch
// row's.  The softmax sums are in 64 bits throughout.  256 batch rows of 4 beams, 9 words: 6 us,
// a launch's latency; the two states behind it (0.8 MB) 3.7.
template <class T, int L>
__global__ __launch_bounds__(256) void beam_small_kernel(BeamArgs a) {
    __shared__ uint64_t s_key[256];
    __shared__ uint32_t s_word[256];                         // what decides between words of one beam of equal scores
    const int W = a.W, V = a.rows.V, per = 256 / L / W;      // batch rows per workgroup
    const int slot = threadIdx.x / L, v = threadIdx.x & (L - 1), mine = slot / W, w = slot - mine * W;
    const int b = blockIdx.x * per + mine;
    const bool in = mine < per && b < a.B;
    const int64_t row = in ? (int64_t)b * W + w : 0;
    const float score = in ? a.scores[row] : 0.f;
    const bool done = in && a.finished[row], dead = !done && score == -INFINITY, word = in && v < V;
    float z = word && !done && !dead ? load1<T>(a.rows.row((int)row), v) : -INFINITY;
    z = z == z ? z : -INFINITY;
    float m = fmaxf(z, -FLT_MAX);
#pragma unroll
    for (int d = L / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, L));
    double s = z == -INFINITY ? 0.0 : exp((double)z - (double)m);
#pragma unroll
    for (int d = L / 2; d; d >>= 1) s += __shfl_xor(s, d, L);
    uint64_t key = 0;
    uint32_t order = 0;
    bool close = false;
    if (word) {
        if (done) key = v == a.pad ? score_key((double)score, 0.0, 0.0) : 0ull;
        else if (dead) key = order_key64(-INFINITY);
        else {
            const double lse = (double)m + log(s);
            key = score_key((double)score, (double)z, lse);
            if (by_logit(score, lse)) {
                // does the next float up or down score the same?  (nothing between them can, if it does not)
                const uint32_t bits = __float_as_uint(z);
                order = order_key(z);
                close = score_key((double)score, (double)__uint_as_float(bits + 1), lse) == key ||
                        score_key((double)score, (double)__uint_as_float(bits - 1), lse) == key;
            }
        }
    }
    s_key[threadIdx.x] = key;
    s_word[threadIdx.x] = order;
    __syncthreads();
    if (!key) return;
    const int first = mine * W * L, i = threadIdx.x - first;
    int place = 0;
    for (int j = 0; j < W * L; ++j) {
        const uint64_t o = s_key[first + j];
        place += o > key || (o == key && j < i) ? 1 : 0;
    }
    if (close) {                         // this beam's words of the same score: by logit (in the loop above: 9.7 us in place of 6)
        for (int j = w * L; j < w * L + L; ++j)
            if (s_key[first + j] == key) place += (s_word[first + j] > order ? 1 : 0) - (s_word[first + j] != order && j < i ? 1 : 0);
    }
    if (place < W) put_beam(a, b, place, key, (uint32_t)w * (uint32_t)V + (uint32_t)v);
}

template <class T>
int launch_small(const BeamArgs &a, hipStream_t stream) {
    const int V = a.rows.V, L = V <= 8 ? 8 : V <= 16 ? 16 : V <= 32 ? 32 : 64;
    const dim3 grid(cdiv(a.B, 256 / L / a.W));
    if (L == 8) hipLaunchKernelGGL((beam_small_kernel<T, 8>), grid, dim3(256), 0, stream, a);
    else if (L == 16) hipLaunchKernelGGL((beam_small_kernel<T, 16>), grid, dim3(256), 0, stream, a);
    else if (L == 32) hipLaunchKernelGGL((beam_small_kernel<T, 32>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((beam_small_kernel<T, 64>), grid, dim3(256), 0, stream, a);
    GSCAN_LAUNCHED("beam_small_kernel");
    return 0;
}

bool small_beams(const gscan_rows &rows) {
    const int L = rows.V <= 8 ? 8 : rows.V <= 16 ? 16 : rows.V <= 32 ? 32 : 64;
    return rows.V <= 64 && rows.inner * L <= 256;
}

struct BeamPlan { int K; TopChunks chunks; };
BeamPlan beam_plan(const gscan_rows &rows) {
    BeamPlan p;
    p.K = (int)std::min<int64_t>(rows.inner, rows.V);
    p.chunks = top_chunks(rows, p.K);
    const int most = std::max(1, kMaxEntries / ((int)rows.inner * p.K));     // the lists of a batch row fit the join's LDS
    if (p.chunks.splits > most) {
        p.chunks.chunk = (cdiv(rows.V, most) + 7) / 8 * 8;
        p.chunks.splits = cdiv(rows.V, p.chunks.chunk);
    }
    return p;
}

// ---- reordering ----
constexpr int kMaxStates = 16;           // per launch: the table travels in the kernel's arguments
constexpr int kSegment = 4096;           // bytes that a wave copies
constexpr int64_t kMaxItems = 1 << 25;   // segments of one state
constexpr int64_t kMaxBlocks = (1 << 24) - 1;      // of a launch, which counts its threads in 32 bits

struct CopyState {
    const char *in; char *out;
    int64_t in_outer, out_outer, in_row, out_row, in_mid, out_mid, bytes;
    int outer, mid, segments, width, first_block;      // width: bytes per access that every address allows
};
struct CopyArgs { int B, W, count; const int32_t *parents; CopyState s[kMaxStates]; };

// The table's pointers are global memory; told so, the copies are global instructions and not flat ones.
template <class U>
__device__ __forceinline__ void copy_segment(const char *in, char *out, int n, int lane, bool zero) {
    typedef const __attribute__((address_space(1))) U *In;
    typedef __attribute__((address_space(1))) U *Out;
    constexpr int R = kSegment / 16 / 64;
    const int words = n / (int)sizeof(U);
    const In src = (In)(uintptr_t)in + lane;
    const Out dst = (Out)(uintptr_t)out + lane;
    int i = 0;
    for (; i + R * 64 <= words; i += R * 64) {
        U x[R];
        if (zero) {
#pragma unroll
            for (int u = 0; u < R; ++u) x[u] = U{};
        } else {
#pragma unroll
            for (int u = 0; u < R; ++u) x[u] = src[i + u * 64];
        }
#pragma unroll
        for (int u = 0; u < R; ++u) dst[i + u * 64] = x[u];
    }
    for (; i + lane < words; i += 64) dst[i] = zero ? U{} : src[i];
}

// A wave per segment of a slice, its four loads before its four stores.  The bytes bind it: 1.07 GB of states written (and
// what of as much is read: parents repeat) in 285 us, where a plain copy of them takes 400 and writing zeros 192.  A wave per
// batch row's segments that reads a parent once for all of its children is slower (307): repeated readings come from the last
// cache.  Segments of 8 KB: 289.
__global__ __launch_bounds__(256) void beam_reorder_kernel(CopyArgs a) {
    int k = 0;
    while (k + 1 < a.count && (int)blockIdx.x >= a.s[k + 1].first_block) ++k;
    const CopyState &s = a.s[k];
    const int lane = threadIdx.x & 63, rows = a.B * a.W;
    const int item = __builtin_amdgcn_readfirstlane(((int)blockIdx.x - s.first_block) * 4 + (int)(threadIdx.x >> 6));
    if (item >= s.outer * rows * s.mid * s.segments) return;
    int q = item / s.segments;
    const int seg = item - q * s.segments;
    const int m = q % s.mid;
    q /= s.mid;
    const int row = q % rows, o = q / rows, b = row / a.W;
    const int parent = __builtin_amdgcn_readfirstlane(a.parents[row]);
    const bool zero = parent < 0 || parent >= a.W;       // nothing is read for it
    const int64_t at = (int64_t)seg * kSegment;
    const char *in = s.in + o * s.in_outer + (int64_t)(b * a.W + (zero ? 0 : parent)) * s.in_row + m * s.in_mid + at;
    char *out = s.out + o * s.out_outer + (int64_t)row * s.out_row + m * s.out_mid + at;
    const int n = (int)min((int64_t)kSegment, s.bytes - at);
    typedef uint32_t Q __attribute__((ext_vector_type(4)));
    switch (s.width) {
        case 16: copy_segment<Q>(in, out, n, lane, zero); break;
        case 8: copy_segment<uint64_t>(in, out, n, lane, zero); break;
        case 4: copy_segment<uint32_t>(in, out, n, lane, zero); break;
        case 2: copy_segment<uint16_t>(in, out, n, lane, zero); break;
        default: copy_segment<uint8_t>(in, out, n, lane, zero); break;
    }
}
}  // namespace

static int check_beams(const gscan_rows &rows) {
    GSCAN_CHECK(rows.inner <= kMaxBeams, "beam_select: %lld beams (1 to %d)", (long long)rows.inner, kMaxBeams);
    GSCAN_CHECK(rows.V <= (1 << 24), "beam_select: %d words (at most 2^24)", rows.V);
    return 0;
}

size_t beam_select_workspace(const gscan_rows &rows) {
    if (check_beams(rows) || small_beams(rows)) return 0;
    const BeamPlan p = beam_plan(rows);
    return (size_t)(rows.outer * rows.inner) * p.chunks.splits * (sizeof(LsePart) + p.K * sizeof(uint64_t));
}

int beam_select(const gscan_rows &rows, const float *scores, const uint8_t *finished, int eos, int pad, float *scores_out,
                int32_t *parents, int64_t *tokens, uint8_t *finished_out, void *workspace, size_t bytes, hipStream_t stream) {
    TRY_RC(check_beams(rows));
    GSCAN_CHECK(scores && finished && scores_out && parents && tokens && finished_out, "beam_select: NULL array");
    GSCAN_CHECK(eos >= 0 && eos < rows.V && pad >= 0 && pad < rows.V, "beam_select: eos %d or pad %d outside the %d words", eos, pad, rows.V);
    GSCAN_CHECK((const void *)scores != (const void *)scores_out && finished != finished_out,
                "beam_select: outputs may not be the inputs");
    BeamArgs a{};
    a.rows = device_rows(rows);
    a.B = (int)rows.outer; a.W = (int)rows.inner; a.eos = eos; a.pad = pad;
    a.scores = scores; a.finished = finished;
    a.scores_out = scores_out; a.parents = parents; a.tokens = tokens; a.finished_out = finished_out;
    if (small_beams(rows))
        return rows.type == GSCAN_F32 ? launch_small<TypeF32>(a, stream) : rows.type == GSCAN_BF16 ? launch_small<TypeBF16>(a, stream)
                                                                                                   : launch_small<TypeF16>(a, stream);
    const size_t need = beam_select_workspace(rows);
    GSCAN_CHECK(workspace && bytes >= need, "beam_select: workspace of %zu bytes, %zu needed", workspace ? bytes : (size_t)0, need);
    GSCAN_CHECK((uintptr_t)workspace % 8 == 0, "beam_select: workspace is not aligned to 8 bytes");
    const BeamPlan p = beam_plan(rows);
    a.K = p.K; a.splits = p.chunks.splits;
    LsePart *parts = (LsePart *)workspace;
    uint64_t *keys = (uint64_t *)(parts + (size_t)a.B * a.W * a.splits);
    a.parts = parts; a.keys = keys;
    TRY_RC(top_chunk_keys(rows, p.K, p.chunks, keys, parts, finished, scores, stream));
    const size_t lists = (size_t)a.W * a.splits, lds = lists * a.K * 12 + lists * 4;
    hipLaunchKernelGGL(beam_join_kernel, dim3(a.B), dim3(256), lds, stream, a);
    GSCAN_LAUNCHED("beam_join_kernel");
    return 0;
}

int beam_reorder(int B, int W, const int32_t *parents, const gscan_state *states, int count, hipStream_t stream) {
    GSCAN_CHECK(B >= 1 && W >= 1 && (int64_t)B * W <= (1 << 24), "beam_reorder: %d batch rows of %d beams", B, W);
    GSCAN_CHECK(parents && states && count >= 1, "beam_reorder: NULL argument or no state");
    for (int k = 0; k < count; ++k) {        // all of them before the first launch
        const gscan_state &t = states[k];
        GSCAN_CHECK(t.in && t.out, "beam_reorder: state %d is NULL", k);
        GSCAN_CHECK(t.outer >= 1 && t.mid >= 1 && t.bytes >= 1 && t.outer <= (1 << 24) && t.mid <= (1 << 24) && t.bytes <= (1ll << 40),
                    "beam_reorder: state %d is empty or too large", k);
        GSCAN_CHECK(t.in_outer >= 0 && t.out_outer >= 0 && t.in_row >= 0 && t.out_row >= 0 && t.in_mid >= 0 && t.out_mid >= 0,
                    "beam_reorder: state %d has a negative stride", k);
        const int64_t items = t.outer * B * W, segments = (t.bytes + kSegment - 1) / kSegment;
        GSCAN_CHECK(items <= kMaxItems && items * t.mid <= kMaxItems && items * t.mid * segments <= kMaxItems,
                    "beam_reorder: state %d has too many pieces", k);
    }
    for (int k = 0; k < count;) {
        CopyArgs a{};
        a.B = B; a.W = W; a.parents = parents;
        int64_t blocks = 0;
        for (; k < count && a.count < kMaxStates; ++k) {
            const gscan_state &t = states[k];
            const int64_t segments = (t.bytes + kSegment - 1) / kSegment, own = (t.outer * B * W * t.mid * segments + 3) / 4;
            if (blocks + own > kMaxBlocks) break;          // a state alone has at most half of them
            CopyState &s = a.s[a.count++];
            s.in = (const char *)t.in; s.out = (char *)t.out;
            s.in_outer = t.in_outer; s.out_outer = t.out_outer; s.in_row = t.in_row; s.out_row = t.out_row;
            s.in_mid = t.in_mid; s.out_mid = t.out_mid; s.bytes = t.bytes;
            s.outer = (int)t.outer; s.mid = (int)t.mid; s.segments = (int)segments;
            const uint64_t all = (uint64_t)(uintptr_t)t.in | (uint64_t)(uintptr_t)t.out | (uint64_t)t.in_outer | (uint64_t)t.out_outer |
                                 (uint64_t)t.in_row | (uint64_t)t.out_row | (uint64_t)t.in_mid | (uint64_t)t.out_mid | (uint64_t)t.bytes;
            s.width = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
            s.first_block = (int)blocks;
            blocks += own;
        }
        hipLaunchKernelGGL(beam_reorder_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
        GSCAN_LAUNCHED("beam_reorder_kernel");
    }
    return 0;
}

}  // namespace gscan
