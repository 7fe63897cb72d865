// A token's choice of experts from its router logits l, over plain rows
// (mixtureofexperts.go:153-205 has the layer's own, csrc/route.hip):
//   s = softmax(l) or logistic(l); order by s + b, or by l itself without biases
//   expert groups: those whose best one or two values sum to most
//   gate_j = scale s_j / (renormalize ? sum over the chosen s : 1)
// the rows in expert order (offsets, tokens, places), and the logits' gradient.
//
// Order.  Without biases experts compare by their logits, as whole numbers of the
// same order; with them by s + b in fp64, because neighbouring fp32 values tie where
// the exact ones do not.  16 lanes (64 above 256 experts) hold a token's experts,
// consecutive ones in a lane.  A round takes their largest key; the first lane
// that has it holds the lowest index.  Keys below every number's: of experts not to
// be chosen (another group's, chosen already: 0 or NaN, which a maximum passes over)
// and above them those that come after all others (logits of -inf and NaN: 1 or -inf;
// places past the last expert too, which the lower indexes keep from being chosen).
//
// Groups.  A group of one, two, four, ... lanes finds its best two by exchanges of
// neighbours, any other through LDS; a group's place is the number of groups
// before it.
//
// Renormalized gates take the chosen scores by their largest, so that neither large nor
// very negative logits leave 0 / 0:  s = e^l, or e^min(l, 0) / (1 + e^-|l|).
// Gates and gradients are taken in fp64 and rounded once (16384 tokens below: 20.8 -> 21.4 us with
// the lists, the gradient's kernel 5.0 -> 6.3; in fp32 with its sums they were off by 2.2 times a
// rounding).
//
// Lists.  A workgroup takes `each` consecutive tokens and writes how often each
// expert was chosen among them; the second kernel adds the counts of the
// workgroups before it and of the experts before, and finds a token's place among
// its workgroup's by a bit mask of tokens per expert.  Nothing depends on the order
// in which anything ran.  Few tokens are one workgroup and one launch.
//
// What bounds it (MI355X): the vector unit and the chain of the rounds; the bytes would
// take 1 us.  16384 tokens x 128 experts, k = 8, sigmoid with biases, 4 of 8 groups by their best
// two: 15.4 us (of some 850 vector instructions per four tokens besides the gates, 235 are the
// scores, 420 the rounds; issue alone would take some 6), lists 6.8 (every workgroup adds the counts of
// all, one wave of it scans, three barriers between).  8192 x 64, k = 4, softmax: 5.3, lists 5.9,
// gradient 4.2.  32 x 64, k = 6, with lists 5.0, one launch.  131072 x 64, k = 6: 22.9, sums before each
// workgroup 5.9, lists 7.1.  16384 x 700, k = 20: 86.5, lists 19.5.  16384 x 60, k = 5, 2 of 5 groups,
// found through LDS: 8.7.
#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace gtmoe {

namespace {

constexpr int kThreads = 256;       // of every kernel but the one that does all
constexpr int kAllThreads = 512;
// Of the first kernel: a workgroup's tokens in one pass of its waves, four waves per SIMD.
constexpr int choose_threads(int experts_per_lane) { return experts_per_lane > 8 ? 512 : 1024; }
constexpr int kMostTokens = 256;    // of one workgroup: four words of a mask
constexpr int kMostExperts = 1024;
constexpr int kMostGroups = 64;
constexpr int kMostHeld = 256;      // workgroups whose counts the second kernel adds itself

// Whole numbers in the order of the values, above 1 for all but NaN.
__device__ __forceinline__ uint32_t order_of(float v)
{
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 as +0
    if (v != v || b == 0xff800000u) return 1;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// The logit a key above 1 stands for.
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <int CTRL>
__device__ __forceinline__ double moved64(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)moved<CTRL>((uint32_t)(b >> 32)) << 32 | moved<CTRL>((uint32_t)b)));
}
template <int CTRL>
__device__ __forceinline__ uint32_t moved64(uint32_t v) { return moved<CTRL>(v); }
__device__ __forceinline__ double lane_value64(double v, int lane)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                            (uint32_t)__builtin_amdgcn_readlane((int)b, lane)));
}
__device__ __forceinline__ double permuted(int from, double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(b >> 32)) << 32 |
                                            (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)b)));
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
__device__ __forceinline__ uint32_t smaller(uint32_t a, uint32_t b) { return min(a, b); }
// (as one instruction each: nothing here is a signalling NaN, which fmax would first quiet.
// No transcendental's result goes in, and the compiler keeps the wait states that DPP
// needs behind whatever wrote its operand.)
__device__ __forceinline__ double larger(double a, double b)
{
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double smaller(double a, double b)
{
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
// keys of what is never chosen, and of what comes last
template <class Key>
struct Never;
template <>
struct Never<uint32_t> {
    static __device__ __forceinline__ uint32_t last() { return 1; }
    static __device__ __forceinline__ uint32_t unless(bool gone, uint32_t k) { return gone ? 0 : k; }
};
template <>
struct Never<double> {
    static __device__ __forceinline__ double last() { return -__builtin_inf(); }
    static __device__ __forceinline__ double unless(bool gone, double k)
    {
        return __hiloint2double(gone ? 0x7ff80000 : __double2hiint(k), __double2loint(k));
    }
};

// e^x for x <= 0 in fp64: powers of two taken out, then the series to r^11 / 11! (below
// 1e-14 of the whole for |r| <= log(2) / 2).
__device__ __forceinline__ double exp64(double x)
{
    x = fmax(x, -750.0);
    const double k = rint(x * 1.4426950408889634);
    double r = fma(k, -6.93147180369123816490e-01, x);  // the first 32 bits of log 2
    r = fma(k, -1.90821492927058770002e-10, r);
    constexpr double inverse[12] = {1.0,       1.0,        1.0 / 2,     1.0 / 6,      1.0 / 24,      1.0 / 120,
                                    1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800};
    double p = inverse[11];
#pragma unroll
    for (int i = 10; i >= 0; --i) p = fma(p, r, inverse[i]);
    return ldexp(p, (int)k);
}
// 1 / d for d of the size of a number of experts at most
__device__ __forceinline__ double inverse64(double d)
{
    double x = __builtin_amdgcn_rcp(d);
    x = fma(fma(-d, x, 1.0), x, x);
    return fma(fma(-d, x, 1.0), x, x);
}
// e^(a - b), a at most b but for NaN, which stays one
__device__ __forceinline__ double exp_between(float a, float b)
{
    const double x = (double)a - (double)b;
    return x != x ? x : exp64(x);
}
__device__ __forceinline__ double logistic64(float l)
{
    const double e = exp64(-fabs((double)l)), r = inverse64(1.0 + e);
    return l != l ? (double)l : l >= 0.f ? r : e * r;
}

// The team's largest key and sums.
template <int TEAM>
__device__ __forceinline__ uint32_t team_largest(uint32_t v)
{
    if constexpr (TEAM == 16) return lanes_max(v, 16);
    return wave_max(v);
}
template <int TEAM>
__device__ __forceinline__ double team_largest(double v)
{
    v = larger(v, moved64<kDppPairs>(v));
    v = larger(v, moved64<kDppFours>(v));
    v = larger(v, moved64<kDppEights>(v));
    v = larger(v, moved64<kDppSixteens>(v));
    if constexpr (TEAM == 64)
        v = larger(larger(lane_value64(v, 0), lane_value64(v, 16)), larger(lane_value64(v, 32), lane_value64(v, 48)));
    return v;
}
template <int TEAM>
__device__ __forceinline__ double team_total(double v)
{
    v += moved64<kDppPairs>(v);
    v += moved64<kDppFours>(v);
    v += moved64<kDppEights>(v);
    v += moved64<kDppSixteens>(v);
    if constexpr (TEAM == 64)
        v = (lane_value64(v, 0) + lane_value64(v, 16)) + (lane_value64(v, 32) + lane_value64(v, 48));
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

// The share s / sum of this lane's choice among the team's, l its logit.
template <int TEAM>
__device__ __forceinline__ double share_of(float l, bool have, bool logistic_scores)
{
    // s = e^upper times a number between 1/2 and 1
    const float upper = logistic_scores && l > 0.f ? 0.f : l;
    float most = team_most<TEAM>(have ? upper : -__builtin_inff());
    if (most == -__builtin_inff()) most = 0.f;  // nothing but -inf: every share is 0
    // (upper is at most `most`; +inf beside itself is NaN)
    double s = exp_between(upper, most);
    if (logistic_scores) s *= inverse64(1.0 + exp64(-fabs((double)l)));
    s = have ? s : 0.0;
    const double sum = team_total<TEAM>(s);
    return sum == 0.0 ? 0.0 : s * inverse64(sum);
}

__device__ __forceinline__ int group_of(int e, uint32_t group_inverse) { return (int)((uint32_t)e * group_inverse >> 22); }

// The best two keys of a group, and merged with another's.
template <class Key>
struct Best {
    Key one = Never<Key>::last(), two = Never<Key>::last();
    __device__ __forceinline__ void add(Key k)
    {
        two = larger(two, smaller(one, k));
        one = larger(one, k);
    }
    template <int CTRL>
    __device__ __forceinline__ void merge()
    {
        const Key o1 = moved64<CTRL>(one), o2 = moved64<CTRL>(two);
        two = larger(smaller(one, o1), larger(two, o2));
        one = larger(one, o1);
    }
};
// What groups compare by: the sum of their best one or two.  Without biases the keys
// are logits': of two, their scores (a softmax's without the common sum).
__device__ __forceinline__ double group_total(const ChooseArgs &a, const Best<double> &b, float)
{
    return a.group_best == 2 && b.two > -__builtin_inf() ? b.one + b.two : b.one;
}
__device__ __forceinline__ double group_total(const ChooseArgs &a, const Best<uint32_t> &b, float most)
{
    if (b.one <= 1) return -__builtin_inf();
    const float l1 = logit_of(b.one), l2 = logit_of(b.two);
    if (a.group_best == 1) return (double)l1;
    double s1 = a.logistic ? logistic64(l1) : exp64((double)l1 - (double)most);
    if (b.two > 1) s1 += a.logistic ? logistic64(l2) : exp64((double)l2 - (double)most);
    return s1;
}

// How groups are found: not at all; as 1, 2, 4, 8 or 16 lanes each; through LDS.
enum GroupForm { kNoGroups = 0, kLaneGroups = 1, kAnyGroups = 2 };
template <class Key, int EPL>
struct WaveGroups {
    Key keys[64 * EPL];
    double total[4][kMostGroups];
    uint8_t allowed[4][kMostGroups];
};
struct NoShared {
};

// tokens [first, last) of the workgroup.  Calls take(t, expert) for each choice.
template <int VALUES, class Key, int TEAM, int EPL, int GROUPS, class Shared, class F>
__device__ __forceinline__ void choose_tokens(const ChooseArgs &a, int first, int last, Shared *shared, F &&take)
{
    constexpr int TEAMS = 64 / TEAM;
    constexpr bool BIASED = sizeof(Key) == 8;
    const int lane = threadIdx.x & 63, in = lane % TEAM, team = lane / TEAM;
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int e0 = in * EPL;
    float b[EPL];
    if constexpr (BIASED) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) b[i] = e0 + i < a.experts ? a.biases[e0 + i] : 0.f;
    }
    for (int t0 = first + wave * TEAMS; t0 < last; t0 += waves * TEAMS) {
        const int t = min(t0 + team, last - 1);  // teams past the last repeat it and keep nothing
        const bool here = t0 + team < last;
        float l[EPL];
        load_logits<VALUES>(l, a.logits, (long long)t * a.ldlogits, e0, a.experts);
        float most = 0.f;  // of a softmax over all experts
        double sum = 0;
        if (!a.logistic && (BIASED || !a.renormalize || GROUPS != kNoGroups)) {
            most = l[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) most = l[i] > most || most != most ? l[i] : most;
            most = team_most<TEAM>(most);
            if (most == -__builtin_inff()) most = 0.f;
            if (!a.renormalize) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) sum += exp_between(l[i], most);
                sum = team_total<TEAM>(sum);
            }
        }
        Key key[EPL];
        if constexpr (BIASED) {
            double s[EPL], inverse = 1.0;
            if (a.logistic) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) s[i] = logistic64(l[i]);
            } else {
                double total = 0;
#pragma unroll
                for (int i = 0; i < EPL; ++i) {
                    s[i] = exp64((double)l[i] - (double)most);
                    total += s[i];
                }
                inverse = inverse64(team_total<TEAM>(total));
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                // (a bias of -inf stays before what comes last)
                key[i] = l[i] > -__builtin_inff() ? larger(fma(s[i], inverse, (double)b[i]), -1e300) : Never<double>::last();
            }
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) key[i] = order_of(l[i]);
        }
        if constexpr (GROUPS == kLaneGroups) {
            Best<Key> best;
#pragma unroll
            for (int i = 0; i < EPL; ++i) best.add(key[i]);
            const int width = a.experts / a.groups / EPL;  // lanes of a group
            if (width > 1) best.template merge<kDppPairs>();
            if (width > 2) best.template merge<kDppFours>();
            if (width > 4) best.template merge<kDppEights>();
            if (width > 8) best.template merge<kDppSixteens>();
            const double mine = group_total(a, best, most);
            const int g = in / width;
            int before = 0;
            for (int o = 0; o < a.groups; o += 4) {
                double other[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) other[i] = permuted(4 * (team * TEAM + (o + i) * width), mine);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    before += o + i < a.groups && (other[i] > mine || (other[i] == mine && o + i < g));
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) key[i] = Never<Key>::unless(before >= a.chosen_groups, key[i]);
        } else if constexpr (GROUPS == kAnyGroups) {
            auto &w = shared[wave];
            Key *keys = w.keys + team * (TEAM * EPL);
#pragma unroll
            for (int i = 0; i < EPL; ++i) keys[e0 + i] = key[i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int each = a.experts / a.groups;
            for (int g = in; g < a.groups; g += TEAM) {
                Best<Key> best;
                for (int i = 0; i < each; ++i) best.add(keys[g * each + i]);
                w.total[team][g] = group_total(a, best, most);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int g = in; g < a.groups; g += TEAM) {
                const double mine = w.total[team][g];
                int before = 0;
                for (int o = 0; o < a.groups; ++o) {
                    const double other = w.total[team][o];
                    before += other > mine || (other == mine && o < g);
                }
                w.allowed[team][g] = before < a.chosen_groups;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                key[i] = Never<Key>::unless(e0 + i >= a.experts || !w.allowed[team][group_of(e0 + i, a.group_inverse)], key[i]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        // choice j is lane j's
        int expert = 0;
        for (int j = 0; j < a.k; ++j) {
            Key top = key[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) top = larger(top, key[i]);
            top = team_largest<TEAM>(top);
            // who has it, one bit a lane; the lowest bit of each team; of that lane the
            // lowest expert (masks of lanes: the scalar unit's work)
            uint64_t has[EPL], who = 0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                has[i] = __ballot(key[i] == top);
                who |= has[i];
            }
            uint64_t first_lanes = who & ~(who - (TEAM == 16 ? 0x0001000100010001ull : 1ull));
            const int winner = __builtin_ctzll(TEAM == 16 ? first_lanes >> (team * (TEAM & 63)) : first_lanes);
            int at = 0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const bool it = __builtin_amdgcn_inverse_ballot_w64(first_lanes & has[i]);
                first_lanes &= ~has[i];
                at = it ? i : at;
                key[i] = Never<Key>::unless(it, key[i]);
            }
            const int e = winner * EPL + __builtin_amdgcn_ds_bpermute(4 * (team * TEAM + winner), at);
            expert = j == in ? e : expert;
        }
        float logit;
        {
            float v[1];
            load_logits<VALUES>(v, a.logits, (long long)t * a.ldlogits, expert, a.experts);
            logit = v[0];
        }
        const bool have = in < a.k;
        double gate;
        if (a.renormalize) gate = share_of<TEAM>(logit, have, a.logistic);
        else gate = a.logistic ? logistic64(logit) : sum == 0.0 ? 0.0 : exp_between(logit, most) * inverse64(sum);
        if (have && here) {
            const long long at = (long long)t * a.k + in;
            a.chosen[at] = expert;
            a.gates[at] = (float)(gate * a.scale);
            take(t, expert);
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

// The place of choice i of the tokens from `first` on, expert e: behind start[e], in the order of
// the tokens, which mask[w][e] has a bit for each.
__device__ __forceinline__ void place(const ChooseArgs &a, int first, int i, int e, const int *start, const unsigned long long *mask)
{
    const int at = i / a.k;
    int to = start[e];
    for (int w = 0; w < at >> 6; ++w) to += __popcll(mask[w * a.experts + e]);
    to += __popcll(mask[(at >> 6) * a.experts + e] & ((1ull << (at & 63)) - 1));
    if (a.rows) a.rows[to] = first + at;
    if (a.places) a.places[(long long)first * a.k + i] = to;
}

template <int VALUES, class Key, int TEAM, int EPL, int GROUPS>
__global__ __launch_bounds__(choose_threads(EPL)) void choose_kernel(ChooseArgs a)
{
    constexpr int THREADS = choose_threads(EPL);
    typedef typename std::conditional<GROUPS == kAnyGroups, WaveGroups<Key, EPL>, NoShared>::type Shared;
    __shared__ Shared shared[GROUPS == kAnyGroups ? THREADS / 64 : 1];
    __shared__ int count[TEAM * EPL];
    for (int e = threadIdx.x; e < TEAM * EPL; e += THREADS) count[e] = 0;
    __syncthreads();
    const int first = blockIdx.x * a.each, last = min(first + a.each, a.tokens);
    choose_tokens<VALUES, Key, TEAM, EPL, GROUPS>(a, first, last, shared, [&](int, int e) { atomicAdd(&count[e], 1); });
    if (!a.counts) return;
    __syncthreads();
    for (int e = threadIdx.x; e < a.ldcounts; e += THREADS)
        a.counts[(long long)blockIdx.x * a.ldcounts + e] = e < a.experts ? (uint16_t)count[e] : (uint16_t)0;
}

// All tokens by one workgroup, lists included.
template <int VALUES, class Key, int TEAM, int EPL, int GROUPS>
__global__ __launch_bounds__(kAllThreads) void choose_all_kernel(ChooseArgs a)
{
    typedef typename std::conditional<GROUPS == kAnyGroups, WaveGroups<Key, EPL>, NoShared>::type Shared;
    __shared__ Shared shared[GROUPS == kAnyGroups ? kAllThreads / 64 : 1];
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
    for (int i = threadIdx.x; i < a.tokens * a.k; i += kAllThreads) place(a, 0, i, a.chosen[i], start, mask);
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

// HELD: the counts of all workgroups are added up here, by as many threads as their
// loads can be in flight together.  The tokens' choices are on their way meanwhile.
constexpr int kPlaceThreads = 1024, kAhead = 2;

template <bool HELD>
__global__ __launch_bounds__(kPlaceThreads) void place_kernel(ChooseArgs a, int blocks)
{
    __shared__ int start[kMostExperts], count[kMostExperts];
    __shared__ unsigned long long mask[kMostTokens / 64 * kMostExperts];
    const int first = blockIdx.x * a.each, last = min(first + a.each, a.tokens);
    const int words = (last - first + 63) >> 6, choices = (last - first) * a.k;
    const int32_t *chosen = a.chosen + (long long)first * a.k;
    int ahead[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
        const int i = threadIdx.x + x * kPlaceThreads;
        ahead[x] = i < choices ? chosen[i] : 0;
    }
    for (int i = threadIdx.x; i < words * a.experts; i += kPlaceThreads) mask[i] = 0;
    for (int e = threadIdx.x; e < a.ldcounts; e += kPlaceThreads) {
        start[e] = HELD ? 0 : a.before[(long long)blockIdx.x * a.ldcounts + e];
        count[e] = HELD ? 0 : a.totals[e];
    }
    int all[8] = {0, 0, 0, 0, 0, 0, 0, 0}, before[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const int columns = a.ldcounts / 8, column = threadIdx.x % columns, row = threadIdx.x / columns, rows = kPlaceThreads / columns;
    if (HELD && row < rows) {
#pragma unroll 4
        for (int b = row; b < blocks; b += rows) {
            const Counts8 c = *reinterpret_cast<const Counts8 *>(a.counts + (long long)b * a.ldcounts + column * 8);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                all[i] += c.n[i];
                before[i] += b < (int)blockIdx.x ? c.n[i] : 0;
            }
        }
    }
    __syncthreads();
    // f(choice of the workgroup, its expert)
    auto each_choice = [&](auto &&f) {
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            const int i = threadIdx.x + x * kPlaceThreads;
            if (i < choices) f(i, ahead[x]);
        }
        for (int i = threadIdx.x + kAhead * kPlaceThreads; i < choices; i += kPlaceThreads) f(i, chosen[i]);
    };
    each_choice([&](int i, int e) {
        const int at = i / a.k;
        atomicOr(&mask[(at >> 6) * a.experts + e], 1ull << (at & 63));
    });
    if (HELD && row < rows) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (all[i]) atomicAdd(&count[column * 8 + i], all[i]);
            if (before[i]) atomicAdd(&start[column * 8 + i], before[i]);
        }
    }
    __syncthreads();
    add_before(start, count, a.experts, blockIdx.x == 0 ? a.offsets : nullptr);
    __syncthreads();
    each_choice([&](int i, int e) { place(a, first, i, e, start, mask); });
}

// A choice outside the experts takes part in nothing.  ALL: every expert has a term (of a softmax
// over all of them), not the chosen alone.
template <int VALUES, int TEAM, int EPL, bool ALL>
__global__ __launch_bounds__(kThreads) void choose_gradient_kernel(ChooseGradientArgs a)
{
    constexpr int TEAMS = 64 / TEAM;
    const int lane = threadIdx.x & 63, in = lane % TEAM, team = lane / TEAM;
    const int e0 = in * EPL;
    const long long step = (long long)gridDim.x * (kThreads / TEAM);
    for (long long t0 = (long long)blockIdx.x * (kThreads / TEAM) + (threadIdx.x >> 6) * TEAMS; t0 < a.tokens; t0 += step) {
        const long long t = min(t0 + team, (long long)a.tokens - 1);
        const bool here = t0 + team < a.tokens;
        int expert = -1;
        float l = 0.f;
        double dg = 0;
        if (in < a.k) {
            expert = a.chosen[t * a.k + in];
            dg = (double)a.gate_gradients[t * a.k + in] * a.scale;
        }
        const bool have = expert >= 0 && expert < a.experts;
        if (have) {
            float v[1];
            load_logits<VALUES>(v, a.logits, t * a.ldlogits, expert, a.experts);
            l = v[0];
        } else {
            expert = -1;
            dg = 0;
        }
        double d;  // what this lane's choice adds to its expert's gradient
        // the choices' terms to those of all experts, and the row
        auto finish = [&](auto (&out)[EPL]) {
            typedef typename std::remove_reference<decltype(out[0])>::type Sum;
            for (int j = 0; j < a.k; ++j) {
                const int from = 4 * (team * TEAM + j);
                const int e = __builtin_amdgcn_ds_bpermute(from, expert);
                Sum v;
                if constexpr (sizeof(Sum) == 8) v = permuted(from, d);
                else v = __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)__float_as_uint((float)d)));
#pragma unroll
                for (int i = 0; i < EPL; ++i)
                    if (e == e0 + i) out[i] += v;
            }
            if (!here) return;
            typedef typename Eight<VALUES>::Store Store;
            Store *p = reinterpret_cast<Store *>(a.logit_gradients) + t * a.ldgradients + e0;
            Store w[EPL];
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const float v = (float)out[i];
                if constexpr (VALUES == kValuesF32) w[i] = v;
                else if constexpr (VALUES == kValuesBf16) w[i] = __builtin_bit_cast(uint16_t, (__bf16)v);
                else w[i] = __builtin_bit_cast(uint16_t, (_Float16)v);
            }
            if (e0 + EPL <= a.experts) {
                __builtin_memcpy(p, w, sizeof w);
            } else {
#pragma unroll
                for (int i = 0; i < EPL; ++i)
                    if (e0 + i < a.experts) p[i] = w[i];
            }
        };
        if constexpr (ALL) {
            float all[EPL], most;
            double out[EPL], sum = 0;
            load_logits<VALUES>(all, a.logits, t * a.ldlogits, e0, a.experts);
            most = all[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) most = all[i] > most || most != most ? all[i] : most;
            most = team_most<TEAM>(most);
            if (most == -__builtin_inff()) most = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                out[i] = exp_between(all[i], most);
                sum += out[i];
            }
            sum = team_total<TEAM>(sum);
            const double inverse = sum == 0.0 ? 0.0 : inverse64(sum);
            d = have ? dg * (exp_between(l, most) * inverse) : 0.0;
            const double by = -team_total<TEAM>(d) * inverse;
#pragma unroll
            for (int i = 0; i < EPL; ++i) out[i] *= by;
            finish(out);
        } else {
            if (a.renormalize) {
                const double share = share_of<TEAM>(l, have, a.logistic);
                const double dot = team_total<TEAM>(have ? share * dg : 0.0);
                d = share * (dg - dot);
                if (a.logistic) d *= logistic64(-l);
            } else {
                d = dg * logistic64(l) * logistic64(-l);
            }
            float out[EPL] = {};  // an expert has one choice's term alone, but for one that stands twice
            finish(out);
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
// Lanes per token, one at least for each choice, and experts per lane.
template <class F>
hipError_t with_team(int experts, int k, F &&f)
{
    if (k > 16) {
        if (experts <= 512) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
        return f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
    }
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
        return with_team(a.experts, a.k, [&](auto team, auto epl) {
            constexpr int V = decltype(v)::value, T = decltype(team)::value, E = decltype(epl)::value;
            const int each = a.experts / a.groups, width = each / E;
            const bool lanes = each % E == 0 && width <= 16 && (width & (width - 1)) == 0;
            auto run = [&](auto key, auto g) {
                typedef decltype(key) K;
                constexpr int G = decltype(g)::value;
                if (all) hipLaunchKernelGGL((choose_all_kernel<V, K, T, E, G>), dim3(1), dim3(kAllThreads), 0, s, a);
                else hipLaunchKernelGGL((choose_kernel<V, K, T, E, G>), dim3(l.blocks), dim3(choose_threads(E)), 0, s, a);
                return hipGetLastError();
            };
            auto with = [&](auto g) { return a.biases ? run(double(), g) : run(uint32_t(), g); };
            if (!grouped) return with(std::integral_constant<int, kNoGroups>());
            return lanes ? with(std::integral_constant<int, kLaneGroups>()) : with(std::integral_constant<int, kAnyGroups>());
        });
    });
    if (e != hipSuccess || !lists || all) return e;
    if (l.blocks <= kMostHeld) {
        hipLaunchKernelGGL(place_kernel<true>, dim3(l.blocks), dim3(kPlaceThreads), 0, s, a, l.blocks);
    } else {
        hipLaunchKernelGGL(count_before_kernel, dim3(l.ldcounts / 8), dim3(kThreads), 0, s, a, l.blocks);
        hipLaunchKernelGGL(place_kernel<false>, dim3(l.blocks), dim3(kPlaceThreads), 0, s, a, l.blocks);
    }
    return hipGetLastError();
}

hipError_t launch_choose_gradient(const ChooseGradientArgs &a, int values, hipStream_t s)
{
    return with_values(values, [&](auto v) {
        return with_team(a.experts, a.k, [&](auto team, auto epl) {
            constexpr int T = decltype(team)::value;
            const int tokens = kThreads / T;
            const unsigned blocks = (unsigned)std::min<long long>(((long long)a.tokens + tokens - 1) / tokens, 1 << 20);
            constexpr int V = decltype(v)::value, E = decltype(epl)::value;
            if (a.renormalize || a.logistic) hipLaunchKernelGGL((choose_gradient_kernel<V, T, E, false>), dim3(blocks), dim3(kThreads), 0, s, a);
            else hipLaunchKernelGGL((choose_gradient_kernel<V, T, E, true>), dim3(blocks), dim3(kThreads), 0, s, a);
            return hipGetLastError();
        });
    });
}

}  // namespace gtmoe
