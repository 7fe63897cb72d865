// A token's choice of experts from its router logits l, over plain rows
// (mixtureofexperts.go:153-205 has the layer's own, csrc/route.hip):
//   s = softmax(l) or logistic(l); order by s + b, or by l itself without biases
//   expert groups: those whose best one or two values sum to most
//   gate_j = scale s_j / (renormalize ? sum over the chosen s : 1)
// the rows in expert order (offsets, tokens, places), and the logits' gradient.
//
// Order.  Values that are compared become whole numbers of the same order: fp32
// logits 32 bits, s + b and sums of two 64 bits of the fp64 value, because
// sums of neighbouring fp32 values tie where the exact ones do not.  A round takes
// the team's largest number; lanes hold consecutive experts, so the first lane
// that has it holds the lowest index.  Keys 0 (not to be chosen: another group,
// already chosen, past the last) and 1 (after everything else: a logit of -inf, a NaN)
// lie below every number's.
//
// Gates come from differences of logarithms of the chosen scores, so that neither
// large nor very negative logits leave 0 / 0:
//   softmax   log s_j - log s_i = l_j - l_i
//   logistic  log s = min(l, 0) - log(1 + e^-|l|)
//
// Lists.  A workgroup takes `each` consecutive tokens and writes how often each
// expert was chosen among them; the second kernel adds the counts of the
// workgroups before it and of the experts before, and finds a token's place among
// its workgroup's by a bit mask of tokens per expert.  Nothing depends on the order
// in which anything ran.  Few tokens are one workgroup and one launch.
#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace gtmoe {

namespace {

constexpr int kThreads = 256;       // of every kernel but the one that does all
constexpr int kAllThreads = 512;
constexpr int kMostTokens = 256;    // of one workgroup: four words of a mask
constexpr int kMostExperts = 1024;
constexpr int kMostChosen = 32;
constexpr int kMostGroups = 64;
constexpr int kMostHeld = 256;      // workgroups whose counts the second kernel adds itself

// Whole numbers in the order of the values, above 1 for all but NaN.
__device__ __forceinline__ uint32_t order_of(float v)
{
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 as +0
    if (v != v || b == 0xff800000u) return 1;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_of(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    if (v != v) return 1;
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double value_of(uint64_t order)
{
    return __longlong_as_double((long long)(order >> 63 ? order & 0x7fffffffffffffffull : ~order));
}

template <int CTRL>
__device__ __forceinline__ uint64_t moved64(uint64_t v)
{
    return (uint64_t)moved<CTRL>((uint32_t)(v >> 32)) << 32 | moved<CTRL>((uint32_t)v);
}
__device__ __forceinline__ uint64_t read64(uint64_t v, int lane)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// The team's largest key and sums.
template <int TEAM>
__device__ __forceinline__ uint32_t team_largest(uint32_t v)
{
    if constexpr (TEAM == 16) return lanes_max(v, 16);
    return wave_max(v);
}
template <int TEAM>
__device__ __forceinline__ uint64_t team_largest(uint64_t v)
{
    v = max(v, moved64<kDppPairs>(v));
    v = max(v, moved64<kDppFours>(v));
    v = max(v, moved64<kDppEights>(v));
    v = max(v, moved64<kDppSixteens>(v));
    if constexpr (TEAM == 64) v = max(max(read64(v, 0), read64(v, 16)), max(read64(v, 32), read64(v, 48)));
    return v;
}
template <int TEAM>
__device__ __forceinline__ float team_total(float v)
{
    if constexpr (TEAM == 16) return sixteen_sum(v);
    return wave_sum(v);
}
template <int TEAM>
__device__ __forceinline__ double team_total(double v)
{
#pragma unroll
    for (int d = 1; d < TEAM; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
template <int TEAM>
__device__ __forceinline__ float team_most(float v)
{
    // by the order of the bits, NaN aside
    const uint32_t o = team_largest<TEAM>(order_of(v));
    return o <= 1 ? -__builtin_inff() : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// EPL consecutive logits of a row from e0 on in fp32; -inf past the last.
template <int VALUES, int EPL>
__device__ __forceinline__ void load_logits(float (&l)[EPL], const void *base, long long at, int e0, int experts)
{
    typedef typename Eight<VALUES>::Store Store;
    const Store *p = reinterpret_cast<const Store *>(base) + at + e0;
    Store w[EPL];
    if (e0 + EPL <= experts) {
        __builtin_memcpy(w, p, sizeof w);
    } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) w[i] = e0 + i < experts ? p[i] : (Store)0;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        float v;
        if constexpr (VALUES == kValuesF32) v = w[i];
        else if constexpr (VALUES == kValuesBf16) v = __uint_as_float((uint32_t)w[i] << 16);
        else v = (float)__builtin_bit_cast(_Float16, w[i]);
        l[i] = e0 + i < experts ? v : -__builtin_inff();
    }
}

// log(logistic(l)) = upper + lower, upper = min(l, 0) exact, lower in (-log 2, 0]
__device__ __forceinline__ float log_logistic_lower(float l) { return -log1pf(exp_minus(l)); }

// The chosen ones' shares s_j / sum, `mine` of the team's slots in this lane: l, whether
// there is one.  Two slots per lane where k exceeds the team.
template <int TEAM, int SLOTS>
__device__ __forceinline__ void shares_of(float (&share)[SLOTS], const float (&l)[SLOTS], const bool (&have)[SLOTS], bool logistic_scores)
{
    float upper[SLOTS], lower[SLOTS], most = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        upper[i] = logistic_scores ? fminf(l[i], 0.f) : l[i];
        if (l[i] != l[i]) upper[i] = l[i];
        lower[i] = logistic_scores ? log_logistic_lower(l[i]) : 0.f;
        if (have[i] && upper[i] > most) most = upper[i];
    }
    most = team_most<TEAM>(most);
    if (most == -__builtin_inff()) most = 0.f;  // nothing but -inf: every share is 0
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        const float d = upper[i] - most;
        // (upper is at most `most`; +inf beside itself is NaN)
        share[i] = have[i] ? exp_minus(d) * (logistic_scores ? expf(lower[i]) : 1.f) : 0.f;
        sum += share[i];
    }
    sum = team_total<TEAM>(sum);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) share[i] = sum == 0.f ? 0.f : share[i] / sum;
}

__device__ __forceinline__ int group_of(int e, uint32_t group_inverse) { return (int)((uint32_t)e * group_inverse >> 22); }

// LDS of a wave for the groups' choice: its tokens' keys and the groups' keys and marks.
template <class Key, int EPL>
struct WaveGroups {
    Key keys[64 * EPL];
    Key best[4][kMostGroups];
    uint32_t allowed[4][kMostGroups];
};
struct NoGroups {
};

// tokens [first, last) of the workgroup.  Calls take(t, slot, expert) for each choice.
template <int VALUES, class Key, int TEAM, int EPL, bool GROUPS, class Shared, class F>
__device__ __forceinline__ void choose_tokens(const ChooseArgs &a, int first, int last, Shared *shared, F &&take)
{
    constexpr int TEAMS = 64 / TEAM, SLOTS = TEAM >= kMostChosen ? 1 : kMostChosen / TEAM;
    constexpr bool WIDE = sizeof(Key) == 8;
    const int lane = threadIdx.x & 63, in = lane % TEAM, team = lane / TEAM;
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int e0 = in * EPL;
    float b[EPL];
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) b[i] = a.biases && e0 + i < a.experts ? a.biases[e0 + i] : 0.f;
    }
    for (int t0 = first + wave * TEAMS; t0 < last; t0 += waves * TEAMS) {
        const int t = min(t0 + team, last - 1);  // teams past the last repeat it and keep nothing
        const bool here = t0 + team < last;
        float l[EPL];
        load_logits<VALUES>(l, a.logits, (long long)t * a.ldlogits, e0, a.experts);
        float most = 0.f, sum = 0.f;  // of a softmax over all experts
        const bool over_all = !a.logistic && (WIDE || !a.renormalize);
        if (over_all) {
            most = l[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) most = l[i] > most || most != most ? l[i] : most;
            most = team_most<TEAM>(most);
            if (most == -__builtin_inff()) most = 0.f;
            if (!a.renormalize) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) sum += exp_minus(l[i] - most);
                sum = team_total<TEAM>(sum);
            }
        }
        Key key[EPL];
        if constexpr (WIDE) {
            double s[EPL], total = 0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                s[i] = a.logistic ? 1.0 / (1.0 + exp(-(double)l[i])) : exp((double)l[i] - (double)most);
                total += s[i];
            }
            if (!a.logistic) {
                total = 1.0 / team_total<TEAM>(total);
#pragma unroll
                for (int i = 0; i < EPL; ++i) s[i] *= total;
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const uint64_t o = order_of(s[i] + (double)b[i]);
                key[i] = e0 + i >= a.experts ? 0 : l[i] != l[i] || l[i] == -__builtin_inff() ? 1 : o;
            }
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) key[i] = e0 + i >= a.experts ? 0 : order_of(l[i]);
        }
        if constexpr (GROUPS) {
            auto &w = shared[wave];
            Key *keys = w.keys + team * (TEAM * EPL);
#pragma unroll
            for (int i = 0; i < EPL; ++i) keys[e0 + i] = key[i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int each = a.experts / a.groups;
            for (int g = in; g < a.groups; g += TEAM) {
                Key one = 0, two = 0;
                for (int i = 0; i < each; ++i) {
                    const Key k = keys[g * each + i];
                    two = k > one ? one : k > two ? k : two;
                    one = k > one ? k : one;
                }
                if constexpr (WIDE)
                    if (a.group_best == 2 && two > 1) one = order_of(value_of(one) + value_of(two));
                w.best[team][g] = one;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int g = in; g < a.groups; g += TEAM) {
                const Key mine = w.best[team][g];
                int before = 0;
                for (int o = 0; o < a.groups; ++o) {
                    const Key k = w.best[team][o];
                    before += k > mine || (k == mine && o < g);
                }
                w.allowed[team][g] = before < a.chosen_groups;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (e0 + i < a.experts && !w.allowed[team][group_of(e0 + i, a.group_inverse)]) key[i] = 0;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        // slot j is lane j % TEAM's
        int expert[SLOTS];
        float logit[SLOTS];
        bool have[SLOTS];
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            expert[i] = 0;
            logit[i] = 0.f;
            have[i] = in + i * TEAM < a.k;
        }
        for (int j = 0; j < a.k; ++j) {
            Key top = key[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) top = max(top, key[i]);
            top = team_largest<TEAM>(top);
            int at = -1;
            float l_at = 0.f;
#pragma unroll
            for (int i = EPL - 1; i >= 0; --i)
                if (key[i] == top) {
                    at = i;
                    l_at = l[i];
                }
            uint64_t who = __ballot(at >= 0);
            if constexpr (TEAM < 64) who = who >> (team * TEAM) & ((1ull << (TEAM & 63)) - 1);
            const int winner = __builtin_ctzll(who);
            const bool won = in == winner;
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (won && i == at) key[i] = 0;
            const int from = 4 * (team * TEAM + winner);
            const int e = __builtin_amdgcn_ds_bpermute(from, e0 + at);
            const float le = __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)__float_as_uint(l_at)));
#pragma unroll
            for (int i = 0; i < SLOTS; ++i)
                if (j == in + i * TEAM) {
                    expert[i] = e;
                    logit[i] = le;
                }
        }
        float gate[SLOTS];
        if (a.renormalize) {
            shares_of<TEAM>(gate, logit, have, a.logistic);
        } else {
#pragma unroll
            for (int i = 0; i < SLOTS; ++i)
                gate[i] = a.logistic ? logistic(logit[i]) : sum == 0.f ? 0.f : exp_minus(logit[i] - most) / sum;
        }
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
            if (have[i] && here) {
                const long long at = (long long)t * a.k + in + i * TEAM;
                a.chosen[at] = expert[i];
                a.gates[at] = gate[i] * a.scale;
                take(t, expert[i]);
            }
    }
}

__device__ __forceinline__ int before_in_wave(int v, int &total)
{
    const int lane = threadIdx.x & 63;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    total = __builtin_amdgcn_readlane(s, 63);
    return s - v;
}

// start[e] += the counts of the experts before e (by wave 0); offsets by the workgroup
// that is told to.
__device__ __forceinline__ void add_before(int *start, const int *count, int experts, int32_t *offsets)
{
    if (threadIdx.x < 64) {
        int before = 0;
        for (int x = 0; x < experts; x += 64) {
            const int e = x + threadIdx.x;
            int total;
            const int at = before + before_in_wave(e < experts ? count[e] : 0, total);
            if (e < experts) {
                start[e] += at;
                if (offsets) offsets[e] = at;
            }
            before += total;
        }
        if (offsets && threadIdx.x == 0) offsets[experts] = before;
    }
}

// The places of tokens [first, last): behind start[e], in the order of the tokens, which
// mask[w][e] has a bit for each.
__device__ __forceinline__ void place_tokens(const ChooseArgs &a, int first, int last, const int *start,
                                             const unsigned long long *mask)
{
    const long long end = (long long)last * a.k;
    for (long long i = (long long)first * a.k + threadIdx.x; i < end; i += blockDim.x) {
        const int t = (int)(i / a.k), e = a.chosen[i], at = t - first;
        int place = start[e];
        for (int w = 0; w < at >> 6; ++w) place += __popcll(mask[w * a.experts + e]);
        place += __popcll(mask[(at >> 6) * a.experts + e] & ((1ull << (at & 63)) - 1));
        if (a.rows) a.rows[place] = t;
        if (a.places) a.places[i] = place;
    }
}

template <int VALUES, class Key, int TEAM, int EPL, bool GROUPS>
__global__ __launch_bounds__(kThreads) void choose_kernel(ChooseArgs a)
{
    typedef typename std::conditional<GROUPS, WaveGroups<Key, EPL>, NoGroups>::type Shared;
    __shared__ Shared shared[GROUPS ? kThreads / 64 : 1];
    __shared__ int count[TEAM * EPL];
    for (int e = threadIdx.x; e < TEAM * EPL; e += kThreads) count[e] = 0;
    __syncthreads();
    const int first = blockIdx.x * a.each, last = min(first + a.each, a.tokens);
    choose_tokens<VALUES, Key, TEAM, EPL, GROUPS>(a, first, last, shared, [&](int, int e) { atomicAdd(&count[e], 1); });
    if (!a.counts) return;
    __syncthreads();
    for (int e = threadIdx.x; e < a.ldcounts; e += kThreads)
        a.counts[(long long)blockIdx.x * a.ldcounts + e] = e < a.experts ? (uint16_t)count[e] : (uint16_t)0;
}

// All tokens by one workgroup, lists included.
template <int VALUES, class Key, int TEAM, int EPL, bool GROUPS>
__global__ __launch_bounds__(kAllThreads) void choose_all_kernel(ChooseArgs a)
{
    typedef typename std::conditional<GROUPS, WaveGroups<Key, EPL>, NoGroups>::type Shared;
    __shared__ Shared shared[GROUPS ? kAllThreads / 64 : 1];
    __shared__ int start[TEAM * EPL], count[TEAM * EPL];
    __shared__ unsigned long long mask[kMostTokens / 64 * TEAM * EPL];
    const int words = (a.tokens + 63) >> 6;
    for (int i = threadIdx.x; i < words * a.experts; i += kAllThreads) mask[i] = 0;
    __syncthreads();
    choose_tokens<VALUES, Key, TEAM, EPL, GROUPS>(a, 0, a.tokens, shared, [&](int t, int e) {
        atomicOr(&mask[(t >> 6) * a.experts + e], 1ull << (t & 63));
    });
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kAllThreads) {
        int n = 0;
        for (int w = 0; w < words; ++w) n += __popcll(mask[w * a.experts + e]);
        count[e] = n;
        start[e] = 0;
    }
    __syncthreads();
    add_before(start, count, a.experts, a.offsets);
    __syncthreads();
    place_tokens(a, 0, a.tokens, start, mask);
}

// Counts of up to eight experts of one workgroup.
struct Counts8 {
    uint16_t n[8];
};

// Where each workgroup's tokens of each expert begin among the expert's, and how
// many the expert has: for more than kMostHeld workgroups.  Eight experts per workgroup.
__global__ __launch_bounds__(kThreads) void count_before_kernel(ChooseArgs a, int blocks)
{
    __shared__ int sums[kThreads][8];
    const int e0 = blockIdx.x * 8;
    const int per = (blocks + kThreads - 1) / kThreads, begin = min((int)threadIdx.x * per, blocks), end = min(begin + per, blocks);
    int n[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int b = begin; b < end; ++b) {
        const Counts8 c = *reinterpret_cast<const Counts8 *>(a.counts + (long long)b * a.ldcounts + e0);
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] += c.n[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[threadIdx.x][i] = n[i];
    __syncthreads();
    if (threadIdx.x < 8) {
        int at = 0;
        for (int x = 0; x < kThreads; ++x) {
            const int v = sums[x][threadIdx.x];
            sums[x][threadIdx.x] = at;
            at += v;
        }
        a.totals[e0 + threadIdx.x] = at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = sums[threadIdx.x][i];
    for (int b = begin; b < end; ++b) {
        const Counts8 c = *reinterpret_cast<const Counts8 *>(a.counts + (long long)b * a.ldcounts + e0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a.before[(long long)b * a.ldcounts + e0 + i] = n[i];
            n[i] += c.n[i];
        }
    }
}

template <bool HELD>
__global__ __launch_bounds__(kThreads) void place_kernel(ChooseArgs a, int blocks)
{
    __shared__ int start[kMostExperts], count[kMostExperts];
    __shared__ unsigned long long mask[kMostTokens / 64 * kMostExperts];
    const int first = blockIdx.x * a.each, last = min(first + a.each, a.tokens);
    const int words = (last - first + 63) >> 6;
    for (int i = threadIdx.x; i < words * a.experts; i += kThreads) mask[i] = 0;
    for (int e = threadIdx.x; e < a.ldcounts; e += kThreads) {
        start[e] = HELD ? 0 : a.before[(long long)blockIdx.x * a.ldcounts + e];
        count[e] = HELD ? 0 : a.totals[e];
    }
    __syncthreads();
    if constexpr (HELD) {
        const int columns = a.ldcounts / 8, column = threadIdx.x % columns;
        int all[8] = {0, 0, 0, 0, 0, 0, 0, 0}, before[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if ((int)threadIdx.x < kThreads / columns * columns) {
#pragma unroll 8
            for (int b = threadIdx.x / columns; b < blocks; b += kThreads / columns) {
                const Counts8 c = *reinterpret_cast<const Counts8 *>(a.counts + (long long)b * a.ldcounts + column * 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    all[i] += c.n[i];
                    before[i] += b < (int)blockIdx.x ? c.n[i] : 0;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (all[i]) atomicAdd(&count[column * 8 + i], all[i]);
                if (before[i]) atomicAdd(&start[column * 8 + i], before[i]);
            }
        }
    }
    const long long end = (long long)last * a.k;
    for (long long i = (long long)first * a.k + threadIdx.x; i < end; i += kThreads) {
        const int at = (int)(i / a.k) - first;
        atomicOr(&mask[(at >> 6) * a.experts + a.chosen[i]], 1ull << (at & 63));
    }
    __syncthreads();
    add_before(start, count, a.experts, blockIdx.x == 0 ? a.offsets : nullptr);
    __syncthreads();
    place_tokens(a, first, last, start, mask);
}

// A choice outside the experts takes part in nothing.
template <int VALUES, int TEAM, int EPL>
__global__ __launch_bounds__(kThreads) void choose_gradient_kernel(ChooseGradientArgs a)
{
    constexpr int TEAMS = 64 / TEAM, SLOTS = TEAM >= kMostChosen ? 1 : kMostChosen / TEAM;
    const int lane = threadIdx.x & 63, in = lane % TEAM, team = lane / TEAM;
    const int e0 = in * EPL;
    const long long step = (long long)gridDim.x * (kThreads / TEAM);
    for (long long t0 = (long long)blockIdx.x * (kThreads / TEAM) + (threadIdx.x >> 6) * TEAMS; t0 < a.tokens; t0 += step) {
        const long long t = min(t0 + team, (long long)a.tokens - 1);
        const bool here = t0 + team < a.tokens;
        int expert[SLOTS];
        float l[SLOTS], dg[SLOTS];
        bool have[SLOTS];
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int j = in + i * TEAM;
            expert[i] = -1;
            dg[i] = l[i] = 0.f;
            if (j < a.k) {
                expert[i] = a.chosen[t * a.k + j];
                dg[i] = a.gate_gradients[t * a.k + j] * a.scale;
            }
            have[i] = expert[i] >= 0 && expert[i] < a.experts;
            if (have[i]) {
                float v[1];
                load_logits<VALUES>(v, a.logits, t * a.ldlogits, expert[i], a.experts);
                l[i] = v[0];
            } else {
                expert[i] = -1;
                dg[i] = 0.f;
            }
        }
        float out[EPL], d[SLOTS];  // d: what slot i adds to its expert's gradient
#pragma unroll
        for (int i = 0; i < EPL; ++i) out[i] = 0.f;
        if (a.renormalize) {
            float share[SLOTS], dot = 0.f;
            shares_of<TEAM>(share, l, have, a.logistic);
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) dot += have[i] ? share[i] * dg[i] : 0.f;
            dot = team_total<TEAM>(dot);
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                d[i] = share[i] * (dg[i] - dot);
                if (a.logistic) d[i] *= logistic(-l[i]);
            }
        } else if (a.logistic) {
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) d[i] = dg[i] * logistic(l[i]) * logistic(-l[i]);
        } else {
            float all[EPL], most, sum = 0.f, dot = 0.f;
            load_logits<VALUES>(all, a.logits, t * a.ldlogits, e0, a.experts);
            most = all[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) most = all[i] > most || most != most ? all[i] : most;
            most = team_most<TEAM>(most);
            if (most == -__builtin_inff()) most = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                out[i] = exp_minus(all[i] - most);
                sum += out[i];
            }
            sum = team_total<TEAM>(sum);
            const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                d[i] = have[i] ? dg[i] * (exp_minus(l[i] - most) * inverse) : 0.f;
                dot += d[i];
            }
            dot = team_total<TEAM>(dot);
#pragma unroll
            for (int i = 0; i < EPL; ++i) out[i] = -dot * (out[i] * inverse);
        }
        for (int j = 0; j < a.k; ++j) {
            const int from = 4 * (team * TEAM + j % TEAM);
            int e = -1;
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i)
                if (j / TEAM == i) {
                    e = expert[i];
                    v = d[i];
                }
            e = __builtin_amdgcn_ds_bpermute(from, e);
            v = __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)__float_as_uint(v)));
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (e == e0 + i) out[i] += v;
        }
        if (!here) continue;
        typedef typename Eight<VALUES>::Store Store;
        Store *p = reinterpret_cast<Store *>(a.logit_gradients) + t * a.ldgradients + e0;
        Store w[EPL];
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            if constexpr (VALUES == kValuesF32) w[i] = out[i];
            else if constexpr (VALUES == kValuesBf16) w[i] = __builtin_bit_cast(uint16_t, (__bf16)out[i]);
            else w[i] = __builtin_bit_cast(uint16_t, (_Float16)out[i]);
        }
        if (e0 + EPL <= a.experts) {
            __builtin_memcpy(p, w, sizeof w);
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (e0 + i < a.experts) p[i] = w[i];
        }
    }
}

template <class F>
hipError_t with_values(int values, F &&f)
{
    switch (values) {
    case kValuesBf16: return f(std::integral_constant<int, kValuesBf16>());
    case kValuesF16: return f(std::integral_constant<int, kValuesF16>());
    default: return f(std::integral_constant<int, kValuesF32>());
    }
}
// Lanes per token and experts per lane.
template <class F>
hipError_t with_team(int experts, F &&f)
{
    if (experts <= 16) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    if (experts <= 64) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
    if (experts <= 128) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
    if (experts <= 256) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 16>());
    if (experts <= 512) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
    return f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

constexpr int kAllTokens = 128;  // up to this many by one workgroup

int tokens_each(int tokens)
{
    // as many workgroups as there are CUs, a round of a workgroup's tokens each at least
    const int each = ((tokens + kMostHeld - 1) / kMostHeld + 15) / 16 * 16;
    return std::max(16, std::min(each, kMostTokens));
}

}  // namespace

ChooseLayout choose_layout(int tokens, int experts)
{
    ChooseLayout l;
    l.each = tokens_each(tokens);
    l.blocks = (tokens + l.each - 1) / l.each;
    l.ldcounts = (experts + 7) / 8 * 8;
    const size_t counts = ((size_t)l.blocks * l.ldcounts * 2 + 15) / 16 * 16;
    l.totals = counts;
    l.before = counts + (size_t)l.ldcounts * 4;
    l.bytes = l.blocks > kMostHeld ? l.before + (size_t)l.blocks * l.ldcounts * 4 : counts;
    if (tokens <= kAllTokens) l.bytes = 0;
    return l;
}

hipError_t launch_choose(ChooseArgs a, int values, void *workspace, hipStream_t s)
{
    const ChooseLayout l = choose_layout(a.tokens, a.experts);
    const bool wide = a.biases || (a.groups > 1 && a.group_best == 2);
    const bool grouped = a.groups > 1 && a.chosen_groups < a.groups;
    const bool lists = a.offsets != nullptr, all = lists && a.tokens <= kAllTokens;
    a.each = l.each;
    a.ldcounts = l.ldcounts;
    a.group_inverse = a.groups > 1 ? (1u << 22) / (uint32_t)(a.experts / a.groups) + 1 : 0;
    if (lists && !all) {
        char *w = reinterpret_cast<char *>(workspace);
        a.counts = reinterpret_cast<uint16_t *>(w);
        a.totals = reinterpret_cast<int *>(w + l.totals);
        a.before = reinterpret_cast<int *>(w + l.before);
    }
    const hipError_t e = with_values(values, [&](auto v) {
        return with_team(a.experts, [&](auto team, auto epl) {
            constexpr int V = decltype(v)::value, T = decltype(team)::value, E = decltype(epl)::value;
            auto run = [&](auto key, auto g) {
                typedef decltype(key) K;
                if (all)
                    hipLaunchKernelGGL((choose_all_kernel<V, K, T, E, decltype(g)::value>), dim3(1), dim3(kAllThreads), 0, s, a);
                else
                    hipLaunchKernelGGL((choose_kernel<V, K, T, E, decltype(g)::value>), dim3(l.blocks), dim3(kThreads), 0, s, a);
                return hipGetLastError();
            };
            if (wide) return grouped ? run(uint64_t(), std::true_type()) : run(uint64_t(), std::false_type());
            return grouped ? run(uint32_t(), std::true_type()) : run(uint32_t(), std::false_type());
        });
    });
    if (e != hipSuccess || !lists || all) return e;
    if (l.blocks <= kMostHeld) {
        hipLaunchKernelGGL(place_kernel<true>, dim3(l.blocks), dim3(kThreads), 0, s, a, l.blocks);
    } else {
        hipLaunchKernelGGL(count_before_kernel, dim3(l.ldcounts / 8), dim3(kThreads), 0, s, a, l.blocks);
        hipLaunchKernelGGL(place_kernel<false>, dim3(l.blocks), dim3(kThreads), 0, s, a, l.blocks);
    }
    return hipGetLastError();
}

hipError_t launch_choose_gradient(const ChooseGradientArgs &a, int values, hipStream_t s)
{
    return with_values(values, [&](auto v) {
        return with_team(a.experts, [&](auto team, auto epl) {
            constexpr int T = decltype(team)::value;
            const int tokens = kThreads / T;
            const unsigned blocks = (unsigned)std::min<long long>(((long long)a.tokens + tokens - 1) / tokens, 1 << 20);
            hipLaunchKernelGGL((choose_gradient_kernel<decltype(v)::value, T, decltype(epl)::value>), dim3(blocks), dim3(kThreads), 0, s, a);
            return hipGetLastError();
        });
    });
}

}  // namespace gtmoe
