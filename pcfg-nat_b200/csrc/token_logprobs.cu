// Log probabilities of given tokens from materialised logits, with the row's entropy and its best alternatives, and the
// gradient of the logits.
//
// With m = max x, S = sum e^(x-m), U = sum e^(x-m) (x-m):  log p_v = (x_v - m) - log S,  H = log S - U / S.
// All three come from one pass over the row: a thread keeps its own m, S and U and rescales them when its maximum grows
// (U' = r (U + S (m - m')), r = e^(m-m'), all terms of one sign), and the threads' triples are joined the same way.
// Entries of -inf (a masked vocabulary) have probability 0 and add nothing; the least finite number of a type is a number
// like any other.  A row with NaN or +inf in it is NaN throughout, a row of nothing but -inf has log p = -inf and H = 0.
//
// The `top` largest values (equal ones by rising index) need no second pass: the top-th largest of the threads' maxima is a
// lower bound of the top-th largest value, so only the few threads whose maximum reaches it look at their numbers again.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "row_vectors.cuh"

namespace cg = cooperative_groups;

namespace pcfgnat {

namespace {

constexpr int kUnroll = 4;            // 16-byte loads of a thread in flight
constexpr int kMaxTop = PCFGNAT_MAX_TOP;
static_assert(kMaxTop <= 32, "a warp writes the alternatives of a row");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFarBelow = -1.0e4f;  // 2^x of anything smaller is 0, and 0 * x stays 0 (with -inf it would be NaN)

struct Stats {
    float m = -FLT_MAX, s = 0.f, u = 0.f;  // maximum of the finite entries, S, and U in units of log 2
};

// Moves the reference of (S, U) from its own maximum up to m.
__device__ __forceinline__ void rescale(Stats &a, float m) {
    const float d = max_nan((a.m - m) * kLog2e, kFarBelow), r = exp2_approx(d);
    a.u = r * (a.u + d * a.s);
    a.s *= r;
    a.m = m;
}
// The triples of a warp's lanes as one, in every lane: one maximum, one rescaling, two sums.
__device__ __forceinline__ Stats join_lanes(Stats a) {
    float m;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(a.m));
    rescale(a, m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
    }
    return a;
}

// One number of a row.
template <bool ENTROPY>
__device__ __forceinline__ void take_one(Stats &a, float x) {
    rescale(a, max_nan(a.m, x));
    const float d = max_nan((x - a.m) * kLog2e, kFarBelow), e = exp2_approx(d);
    a.s += e;
    if (ENTROPY) a.u += e * d;
}

// kUnroll vectors of a row: one maximum and one rescaling for all, then two numbers at a time.
template <typename T, bool ENTROPY>
__device__ __forceinline__ void take(Stats &a, const uint4 (&raw)[kUnroll]) {
    constexpr int kWords = 4 * kUnroll;
    uint32_t word[kWords];
#pragma unroll
    for (int k = 0; k < kUnroll; k++) {
        word[4 * k] = raw[k].x, word[4 * k + 1] = raw[k].y, word[4 * k + 2] = raw[k].z, word[4 * k + 3] = raw[k].w;
    }
    rescale(a, max_nan(a.m, max_of_words<T, kWords>(word)));
    const Packed minus_m(-a.m, -a.m), log2e(kLog2e, kLog2e);
    Packed s(0.f, 0.f), u(0.f, 0.f);
    constexpr int kStep = sizeof(T) == 4 ? 2 : 1;
#pragma unroll
    for (int k = 0; k < kWords; k += kStep) {
        const Packed y = (pair_of_words<T>(word, k) + minus_m) * log2e;
        float2 d = y.get();
        if (ENTROPY) d.x = max_nan(d.x, kFarBelow), d.y = max_nan(d.y, kFarBelow);
        const Packed e(exp2_approx(d.x), exp2_approx(d.y));
        s = s + e;
        if (ENTROPY) u = fma(e, Packed(d.x, d.y), u);
    }
    const float2 s2 = s.get(), u2 = u.get();
    a.s += s2.x + s2.y;
    if (ENTROPY) a.u += u2.x + u2.y;
}

// Order-preserving integers of floats (no NaN among them).
__device__ __forceinline__ uint32_t rank_bits(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);  // -0 equals +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// One key per entry: larger value first, then smaller index.  No entry has key 0.
__device__ __forceinline__ uint64_t entry_key(float x, int index) {
    return (uint64_t)rank_bits(x) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float rank_value(uint32_t b) { return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b); }
__device__ __forceinline__ float key_value(uint64_t k) { return rank_value((uint32_t)(k >> 32)); }
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

struct Rows {
    const void *logits;
    int64_t inner, stride_outer, stride_inner;  // row r lies at (r / inner) * stride_outer + (r % inner) * stride_inner
    int V;
    template <typename T>
    __device__ __forceinline__ const T *at(int64_t r) const {
        const T *p = static_cast<const T *>(logits);
        if (r < inner) return p + r * stride_inner;  // all rows at one stride: no division
        const uint32_t outer = (uint32_t)r / (uint32_t)inner, rest = (uint32_t)r - outer * (uint32_t)inner;
        return p + outer * stride_outer + rest * stride_inner;
    }
};

struct Given {
    const int64_t *tokens;
    int64_t ignore;
    int has_ignore;
};

struct Results {
    int top;
    float *logprob, *entropy, *top_logprob;
    int64_t *top_index;
    float *kept;
    int *status;
};

// The numbers of a row that one team of threads looks at.
template <typename T>
struct Part {
    const T *row;
    const uint4 *vec;
    int head, first, last;  // vectors [first, last)
    int loose, vecs;        // numbers in no vector that this part takes, vectors of the whole row
    __device__ __forceinline__ int loose_at(int i) const { return i < head ? i : i + vecs * RowCut<T>::kVec; }
    __device__ __forceinline__ Part(const Rows &rows, int64_t r, int rank, int parts) {
        row = rows.at<T>(r);
        const RowCut<T> cut(row, rows.V);
        head = cut.head, vecs = cut.vecs;
        vec = reinterpret_cast<const uint4 *>(row + cut.head);
        const int share = (cut.vecs + parts - 1) / parts;
        first = min(rank * share, cut.vecs), last = min(first + share, cut.vecs);
        loose = rank == 0 ? cut.loose(rows.V) : 0;
    }
    // kUnroll vectors from number i on, NT apart; nothing but -inf behind the last.
    template <int NT>
    __device__ __forceinline__ void load(uint4 (&raw)[kUnroll], int i) const {
#pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            const uint32_t none = neg_inf_word<T>();
            raw[k] = i + k * NT < last ? __ldg(vec + i + k * NT) : make_uint4(none, none, none, none);
        }
    }
};

// What a team of NT threads shares.
template <int NT>
struct Team {
    static constexpr int kWarps = NT / 32;
    static constexpr int kCandidates = NT == 32 ? 128 : 512;  // values that reach the bound; more are found one at a time
    Stats part[kWarps];
    uint32_t maxima[NT];
    uint16_t again[NT];  // threads whose numbers are looked at once more
    uint64_t found[kCandidates];
    uint64_t best[kMaxTop];
    Stats whole;
    int n_found, n_again;
    uint32_t bound;
};

template <int NT>
__device__ __forceinline__ void team_sync() {
    if (NT == 32) __syncwarp();
    else __syncthreads();
}

// The top-th largest of the threads' maxima, by one warp; 0 where fewer threads saw anything: every number is a candidate.
template <int NT>
__device__ __forceinline__ uint32_t lower_bound_of_top(const Team<NT> &t, int top, int lane) {
    constexpr int kWarps = Team<NT>::kWarps;
    uint32_t v[kWarps], best = 0, at = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) v[w] = t.maxima[w * 32 + lane], best = max(best, v[w]);
    for (int k = 0; k < top; k++) {
        at = __reduce_max_sync(0xffffffffu, best);
        if (at == 0) break;
        const uint32_t who = __ballot_sync(0xffffffffu, best == at);
        if (lane == __ffs(who) - 1) {
            bool gone = false;
            best = 0;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                if (!gone && v[w] == at) v[w] = 0, gone = true;
                best = max(best, v[w]);
            }
        }
    }
    return at;
}

// The `top` best entries of a part, sorted, into t.best (zeroed before; they stay 0 where there are fewer).
template <typename T, int NT>
__device__ __forceinline__ void best_entries(Team<NT> &t, const Part<T> &p, int top, uint32_t own_max, int tid) {
    constexpr int kVec = RowCut<T>::kVec, kWarps = Team<NT>::kWarps;
    const int warp = tid >> 5, lane = tid & 31;
    const uint32_t least = t.bound;
    const float at_least = least ? rank_value(least) : neg_inf();
    const auto offer = [&](float x, int index) {
        if (x == neg_inf() || !(x >= at_least)) return;
        const int at = atomicAdd(&t.n_found, 1);
        if (at < Team<NT>::kCandidates) t.found[at] = entry_key(x, index);
    };
    const auto offer_vector = [&](const uint4 &raw, int i) {
        const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
        if (!(max_of_words<T, 4>(word) >= at_least)) return;  // as in most vectors
        float x[kVec];
        unpack_vec<T, kVec>(raw, x);
#pragma unroll
        for (int j = 0; j < kVec; j++) offer(x[j], p.head + i * kVec + j);
    };
    if (own_max != 0 && own_max >= least) t.again[atomicAdd(&t.n_again, 1)] = (uint16_t)tid;
    team_sync<NT>();
    // thread by thread of those, vector by vector, dealt out to all threads of the team
    const int each = (p.last - p.first + NT - 1) / NT, items = t.n_again * each;
    for (int i0 = tid; i0 < items; i0 += kUnroll * NT) {
        uint4 raw[kUnroll];
        int at[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            const int item = i0 + k * NT, which = item / each;
            at[k] = item < items ? p.first + t.again[which] + (item - which * each) * NT : p.last;
            if (at[k] < p.last) raw[k] = __ldg(p.vec + at[k]);
        }
#pragma unroll
        for (int k = 0; k < kUnroll; k++)
            if (at[k] < p.last) offer_vector(raw[k], at[k]);
    }
    for (int i = tid; i < p.loose; i += NT) offer(num_to_float<T>(p.row[p.loose_at(i)]), p.loose_at(i));
    team_sync<NT>();
    const int n = t.n_found;
    if (n <= Team<NT>::kCandidates) {
        for (int i = tid; i < n; i += NT) {
            const uint64_t key = t.found[i];
            int better = 0;
            for (int j = 0; j < n; j++) better += t.found[j] > key;
            if (better < top) t.best[better] = key;
        }
        return;
    }
    // Many equal values at the bound, or few threads that saw any: one sweep over the part per alternative.
    uint64_t last = ~0ull;
    for (int k = 0; k < top; k++) {
        uint64_t best = 0;
        const auto look = [&](float x, int index) {
            const uint64_t key = entry_key(x, index);
            if (x != neg_inf() && key < last && key > best) best = key;
        };
        for (int i = p.first + tid; i < p.last; i += NT) {
            float x[kVec];
            unpack_vec<T, kVec>(__ldg(p.vec + i), x);
#pragma unroll
            for (int j = 0; j < kVec; j++) look(x[j], p.head + i * kVec + j);
        }
        if (tid < p.loose) look(num_to_float<T>(p.row[p.loose_at(tid)]), p.loose_at(tid));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        team_sync<NT>();
        if (lane == 0) t.found[warp] = best;
        team_sync<NT>();
        for (int w = 0; w < kWarps; w++) best = t.found[w] > best ? t.found[w] : best;
        if (tid == 0) t.best[k] = best;
        last = best;
    }
}

__device__ __forceinline__ void leave_out(const Results &out, int64_t r, int tid) {
    if (tid == 0) {
        out.logprob[r] = 0.f;
        if (out.entropy) out.entropy[r] = 0.f;
        if (out.kept) out.kept[2 * r] = out.kept[2 * r + 1] = 0.f;
    }
    if (tid < out.top) out.top_logprob[r * out.top + tid] = 0.f, out.top_index[r * out.top + tid] = -1;
}

// The end of a row, by one warp: `a` is the whole row's, x its number at the given token.
template <int NT, bool ENTROPY>
__device__ __forceinline__ void write_out(const Results &out, const Team<NT> &t, const Stats &a, int64_t r, bool inside, float x,
                                          int lane) {
    const float log_s = logf(a.s);  // -inf for a row of nothing but -inf
    const int top = out.top;
    if (lane == 0) {
        if (!inside) flag(out.status, PCFGNAT_STATUS_BAD_INDEX);
        out.logprob[r] = !inside ? CUDART_NAN_F : a.s == 0.f ? neg_inf() : (x - a.m) - log_s;
        if (ENTROPY) out.entropy[r] = a.s == 0.f ? 0.f : log_s - kLn2 * (a.u / a.s);
        if (out.kept) out.kept[2 * r] = a.m, out.kept[2 * r + 1] = log_s;
    }
    if (lane < top) {
        const uint64_t key = a.s > 0.f ? t.best[lane] : 0;
        // a row that is no distribution is NaN; an alternative that does not exist has no probability
        out.top_logprob[r * top + lane] = key ? (key_value(key) - a.m) - log_s : a.s >= 0.f ? neg_inf() : CUDART_NAN_F;
        out.top_index[r * top + lane] = key ? key_index(key) : -1;
    }
}

// What every thread found of its part: the whole part's in warp 0, and what the search for alternatives starts from.
template <int NT>
__device__ __forceinline__ Stats join_team(Team<NT> &t, Stats a, uint32_t own_max, int top, int tid) {
    const int warp = tid >> 5, lane = tid & 31;
    if (top) t.maxima[tid] = own_max;
    a = join_lanes(a);
    if (Team<NT>::kWarps > 1 && lane == 0) t.part[warp] = a;
    team_sync<NT>();
    if (warp == 0) {
        if (Team<NT>::kWarps > 1) a = join_lanes(lane < Team<NT>::kWarps ? t.part[lane] : Stats());
        if (top) {
            const uint32_t least = a.s > 0.f ? lower_bound_of_top<NT>(t, top, lane) : 0xffffffffu;  // that many or none
            if (lane == 0) t.bound = least, t.n_found = t.n_again = 0;
            t.best[lane] = 0;
        }
    }
    return a;
}
// 0: no entry but -inf (or NaN, where nothing is chosen)
__device__ __forceinline__ uint32_t maximum_of(const Stats &a) { return a.s > 0.f ? rank_bits(a.m) : 0u; }

// Blocks that fit an SM.  More hide more of the memory's latency until their registers run out: with 40 000 numbers a row,
// float32 rows 61, 51 and 56 us with 9, 10 and 12 blocks, halves 57, 57 and 60 us for 2 272 rows with eight alternatives.
template <typename T, int NT>
constexpr int kResident = NT == 256 ? 4 : NT == 64 ? 16 : NT == 32 || sizeof(T) == 4 ? 10 : 9;

// A team of NT threads per row or, in a cluster, per part of a row; the first block of a cluster joins the parts.
template <typename T, int NT, bool ENTROPY>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT, kResident<T, NT>)
    token_logprobs_kernel(Rows rows, int64_t n_rows, Given given, Results out) {
    constexpr int kTeams = NT == 32 ? 4 : 1;
    __shared__ Team<NT> teams[kTeams];
    Team<NT> &t = teams[kTeams == 1 ? 0 : threadIdx.x / NT];
    const int tid = threadIdx.x % NT, warp = tid >> 5, lane = tid & 31;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = kTeams == 1 ? (int)cluster.num_blocks() : 1, rank = kTeams == 1 ? (int)cluster.block_rank() : 0;
    const int64_t r = kTeams == 1 ? (int64_t)(blockIdx.x / (unsigned)parts) : (int64_t)blockIdx.x * kTeams + threadIdx.x / NT;
    if (r >= n_rows) return;
    const int top = out.top;
    const int64_t token = given.tokens[r];
    if (given.has_ignore && token == given.ignore) {
        if (rank == 0) leave_out(out, r, tid);
        return;
    }
    const Part<T> p(rows, r, rank, parts);
    const bool inside = token >= 0 && token < rows.V;
    const float x_token = tid == 0 && inside ? num_to_float<T>(p.row[token]) : 0.f;  // needed at the end, on its way from here on
    Stats a;
    for (int i = p.first + tid; i < p.last; i += kUnroll * NT) {
        uint4 raw[kUnroll];
        p.template load<NT>(raw, i);
        take<T, ENTROPY>(a, raw);
    }
    if (tid < p.loose) take_one<ENTROPY>(a, num_to_float<T>(p.row[p.loose_at(tid)]));
    const uint32_t own_max = maximum_of(a);
    a = join_team<NT>(t, a, own_max, top, tid);
    if (top) {
        team_sync<NT>();
        best_entries<T, NT>(t, p, top, own_max, tid);
        team_sync<NT>();
    }
    if (parts > 1) {
        if (tid == 0) t.whole = a;
        cluster.sync();
        if (rank == 0) {
            if (warp == 0) a = join_lanes(lane < parts ? *cluster.map_shared_rank(&t.whole, lane) : Stats());
            if (top) {  // the parts' best entries side by side
                for (int i = tid; i < parts * top; i += NT) t.found[i] = cluster.map_shared_rank(t.best, i / top)[i % top];
                __syncthreads();
                if (tid < top) t.best[tid] = 0;
            }
        }
        cluster.sync();  // a block's memory is there until it has been read
        if (rank) return;
        if (top) {
            for (int i = tid; i < parts * top; i += NT) {
                const uint64_t key = t.found[i];
                int better = 0;
                for (int j = 0; j < parts * top; j++) better += t.found[j] > key;
                if (key && better < top) t.best[better] = key;
            }
            __syncthreads();
        }
    }
    if (warp == 0) write_out<NT, ENTROPY>(out, t, a, r, inside, x_token, lane);
}

// d x_v = p_v (-G - h (log p_v + H)) + sum of the gradients given to v, G their sum over the row, h the entropy's.
// The few entries that tokens and alternatives name are formed again, with what is added, before they are rounded.
// A team of NT threads per row, or per part of a row (blockIdx.y) where the rows alone do not fill the GPU.
template <typename T, int NT>
constexpr int kGradAhead = NT == 512 && sizeof(T) == 2 ? 2 : 4;  // loads of a thread in flight
template <typename T, int NT>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT, NT < 512 ? 12 : sizeof(T) == 2 ? 4 : 3)
    token_logprobs_grad_kernel(Rows rows, int64_t n_rows, Given given, int top, const float *__restrict__ kept,
                               const float *__restrict__ entropy, const int64_t *__restrict__ top_index,
                               const float *__restrict__ g_logprob, const float *__restrict__ g_entropy,
                               const float *__restrict__ g_top, T *dlogits, int64_t pitch, int *status) {
    constexpr int kVec = RowCut<T>::kVec, kAhead = kGradAhead<T, NT>, kTeams = NT == 32 ? 4 : 1;
    __shared__ int all_at[kTeams][kMaxTop + 1];
    __shared__ float all_add[kTeams][kMaxTop + 1];
    const int tid = threadIdx.x % NT, team = kTeams == 1 ? 0 : threadIdx.x / NT;
    int *at = all_at[team];
    float *add = all_add[team];
    const int64_t r = (int64_t)blockIdx.x * kTeams + team;
    if (r >= n_rows) return;
    const int V = rows.V;
    const T *row = rows.at<T>(r);
    T *out = dlogits + r * pitch;
    const int64_t token = given.tokens[r];
    const bool left_out = given.has_ignore && token == given.ignore;
    const float m = kept[2 * r], log_s = kept[2 * r + 1];
    const bool bad = !left_out && g_logprob && (token < 0 || token >= V);
    if (bad && tid == 0) flag(status, PCFGNAT_STATUS_BAD_INDEX);
    for (int k = tid; k <= top; k += NT) {  // number 0: the token
        int64_t index = -1;
        float g = 0.f;
        if (k == 0 && g_logprob) index = token, g = g_logprob[r];
        if (k > 0 && g_top) index = top_index[r * top + k - 1], g = index < 0 ? 0.f : g_top[r * top + k - 1];
        at[k] = index < 0 || index >= V ? -1 : (int)index;
        add[k] = g;
    }
    team_sync<NT>();
    float G = 0.f;
    for (int k = 0; k <= top; k++) G += add[k];
    if (bad) G = CUDART_NAN_F;
    const float h = g_entropy ? g_entropy[r] : 0.f, H = g_entropy ? entropy[r] : 0.f;
    const bool zero = left_out || log_s == neg_inf();  // not asked for, or nothing in it
    const float base = -G - h * H;
    const auto grad = [&](float x) {
        const float lp = max_nan((x - m) - log_s, kFarBelow);
        return exp2_approx(lp * kLog2e) * (base - h * lp);
    };
    const Packed minus_m(-m, -m), minus_log_s(-log_s, -log_s), log2e(kLog2e, kLog2e), base2(base, base), minus_h(-h, -h);
    const auto grad_vec = [&](const uint4 &raw) {
        uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int k = 0; k < 4; k += sizeof(T) == 4 ? 2 : 1) {
            float2 lp = (pair_of_words<T>(word, k) + minus_m + minus_log_s).get();
            lp.x = max_nan(lp.x, kFarBelow), lp.y = max_nan(lp.y, kFarBelow);
            const Packed lp2(lp.x, lp.y);
            const float2 y = (lp2 * log2e).get();
            const float2 d = (Packed(exp2_approx(y.x), exp2_approx(y.y)) * fma(minus_h, lp2, base2)).get();
            if constexpr (sizeof(T) == 4) word[k] = __float_as_uint(d.x), word[k + 1] = __float_as_uint(d.y);
            else word[k] = pack_vec<T, 2>({d.x, d.y});
        }
        return make_uint4(word[0], word[1], word[2], word[3]);
    };
    const RowCut<T> cut(out, V);
    const bool same = !((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15);
    // this block's part: vectors [first, last), with the numbers in no vector in the first one
    const int share = (cut.vecs + gridDim.y - 1) / gridDim.y;
    const int first = min((int)blockIdx.y * share, cut.vecs), last = min(first + share, cut.vecs);
    if (tid < (blockIdx.y == 0 ? cut.loose(V) : 0)) {
        const int i = cut.loose_at(tid);
        out[i] = num_from_float<T>(zero ? 0.f : grad(num_to_float<T>(row[i])));
    }
    uint4 *to = reinterpret_cast<uint4 *>(out + cut.head);
    if (zero) {
        for (int i = first + tid; i < last; i += NT) to[i] = make_uint4(0, 0, 0, 0);
        return;
    }
    if (same) {
        const uint4 *vec = reinterpret_cast<const uint4 *>(row + cut.head);
        int i = first + tid;
        for (; i + (kAhead - 1) * NT < last; i += kAhead * NT) {
            uint4 raw[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) raw[k] = __ldg(vec + i + k * NT);
#pragma unroll
            for (int k = 0; k < kAhead; k++) to[i + k * NT] = grad_vec(raw[k]);
        }
        for (; i < last; i += NT) to[i] = grad_vec(__ldg(vec + i));
    } else {  // rows that begin at different places of a 16-byte vector
        for (int i = first * kVec + tid; i < last * kVec; i += NT)
            out[cut.head + i] = num_from_float<T>(grad(num_to_float<T>(row[cut.head + i])));
    }
    team_sync<NT>();
    for (int q = tid; q <= top; q += NT) {
        if (at[q] < 0) continue;
        const int i = at[q], v = i < cut.head || i >= cut.head + cut.vecs * kVec ? -1 : (i - cut.head) / kVec;
        if (v < 0 ? blockIdx.y == 0 : v >= first && v < last) {  // written by this block
            float g = 0.f;
            for (int k = 0; k <= top; k++) g += at[k] == i ? add[k] : 0.f;
            out[i] = num_from_float<T>(grad(num_to_float<T>(row[i])) + g);
        }
    }
}

}  // namespace

int launch_token_logprobs(const void *logits, int dtype, int64_t n, int64_t inner, int64_t stride_outer, int64_t stride_inner, int V,
                          const int64_t *tokens, int has_ignore, int64_t ignore, int top, float *logprob, float *entropy,
                          float *top_logprob, int64_t *top_index, float *kept, int *status, cudaStream_t st) {
    if (n == 0) return PCFGNAT_OK;
    const Rows rows{logits, inner, stride_outer, stride_inner, V};
    const Given given{tokens, ignore, has_ignore};
    const Results out{top, logprob, entropy, top_logprob, top_index, kept, status};
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t vecs = V / RowCut<T>::kVec, sms = sm_count();
        const auto run = [&](auto team, int parts) {
            constexpr int NT = decltype(team)::value;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)(NT == 32 ? (n * NT + 127) / 128 : n * parts));
            cfg.blockDim = dim3(NT == 32 ? 128 : NT);
            cfg.stream = st;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = (unsigned)parts;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = parts > 1 ? 1 : 0;
            return cuda_rc(entropy ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, NT, true>, rows, n, given, out)
                                   : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, NT, false>, rows, n, given, out));
        };
        // A warp per row while a lane has no more than eight vectors.  Where many rows keep every SM busy a block of 64 (2 000 rows of
        // 4 096 halves 14.4 against 17.4 us by 128) or 128 threads; 128 too where a row is over in a few loads.  For fewer rows one
        // of 256 (64 rows of 40 000 halves 8.2 against 10.2 us), and up to eight of them where a thread would see more than twenty
        // vectors (64 rows of 128 256: 14.3 against 18.4 us) while that is no more than the GPU holds: a cluster costs two barriers
        // (64 rows of 40 000 halves by clusters of two 10.2 us).
        if (vecs <= 256) return run(std::integral_constant<int, 32>(), 1);
        if (n > 2 * sms && vecs <= 1024) return run(std::integral_constant<int, 64>(), 1);
        if (n > 2 * sms || vecs <= 1024) return run(std::integral_constant<int, 128>(), 1);
        int parts = 1;
        while (parts < 8 && vecs > (int64_t)parts * 20 * 256 && n * parts * 2 <= 2 * sms) parts *= 2;
        return run(std::integral_constant<int, 256>(), parts);
    });
}

int launch_token_logprobs_grad(const void *logits, int dtype, int64_t n, int64_t inner, int64_t stride_outer, int64_t stride_inner,
                               int V, const int64_t *tokens, int has_ignore, int64_t ignore, int top, const float *kept,
                               const float *entropy, const int64_t *top_index, const float *g_logprob, const float *g_entropy,
                               const float *g_top, void *dlogits, int64_t pitch, int *status, cudaStream_t st) {
    if (n == 0) return PCFGNAT_OK;
    const Rows rows{logits, inner, stride_outer, stride_inner, V};
    const Given given{tokens, ignore, has_ignore};
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        // A warp per row while a lane has no more than eight vectors, blocks of 128 threads up to 32 KB a row, else of 512: rows of
        // 1 000 halves 16.5 us by warps and 22.6 by blocks, of 40 000 halves 274 and 295 us by blocks of 512 and 128 threads.
        const int64_t vecs = V / RowCut<T>::kVec;
        const auto run = [&](auto team) {
            constexpr int NT = decltype(team)::value;
            // parts of at least two vectors per thread while there are fewer threads than the GPU holds at once
            const int64_t room = 2048 / NT * (int64_t)sm_count() / n;
            const int64_t parts = NT == 32 ? 1 : std::max<int64_t>(1, std::min<int64_t>({room, vecs / (2 * NT), 64}));
            token_logprobs_grad_kernel<T, NT><<<dim3((unsigned)(NT == 32 ? (n * NT + 127) / 128 : n), (unsigned)parts), NT == 32 ? 128 : NT, 0, st>>>(
                rows, n, given, top, kept, entropy, top_index, g_logprob, g_entropy, g_top, static_cast<T *>(dlogits), pitch, status);
            return cuda_rc(cudaGetLastError());
        };
        if (vecs <= 256) return run(std::integral_constant<int, 32>());
        if (vecs <= 2048) return run(std::integral_constant<int, 128>());
        return run(std::integral_constant<int, 512>());
    });
}

}  // namespace pcfgnat
