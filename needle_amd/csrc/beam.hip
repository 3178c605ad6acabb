// One step of a beam search: the k best continuations over the beams of every group, and the move of what the beams
// carry to their picks' places.
//
//   total(b, t) = scores[b] + x[b][t] - lse[b],   lse[b] = log sum_t exp x[b][t] over the admitted t (0 without normalize)
//
// lse is one number per row, so within a row the order of the totals is the order of the logits: one pass over the logits
// keeps, per piece of a row, its maximum, its sum of exponentials and its k largest logits; a second, small kernel joins the
// pieces of a group.  The pass is bound by the bytes of the logits.
//
// Picks are whole numbers and two beams' totals may lie a rounding apart, so all that decides between beams is held in 64
// bits: the exponentials (a few units in the last place each), their sums, the totals.  A sum is held in units of its largest
// term, which so adds exactly 1: a row of which one continuation counts has the logarithm of 1, and its total is its score, as
// an ended beam's is.
#include "nh_values.h"

namespace nh {

constexpr uint32_t BEAM_K_MAX = 256, BEAMS_MAX = 1024;
constexpr uint32_t PIECE_THREADS = 256;

// ---- exponential of x <= 0 in 64 bits --------------------------------------------------------
// exp x = 2^n 2^f with n the whole number nearest to x / ln 2 (found by adding 1.5 * 2^52, which leaves it in the low
// bits of the sum), |f| <= 1/2, and 2^f = 1 + f g(f) with g interpolated at eleven Chebyshev nodes: 2e-17 of the result
// off besides the roundings, and exactly 1 at 0.  Below -700 the result is that of -700, 1e-304: nothing beside a 1.
constexpr double ONE_AND_A_HALF = 6755399441055744.0, PER_LN2 = 1.4426950408889634074;
__device__ inline double add_to_high(double d, int n) { return __hiloint2double(__double2hiint(d) + n, __double2loint(d)); }
__device__ inline double exp2_near_0(double f) {
    double g = 0x1.e9d3fe3952179p-32;
    g = __builtin_fma(g, f, 0x1.e6063f7217bc6p-28);
    g = __builtin_fma(g, f, 0x1.b524fae627834p-24);
    g = __builtin_fma(g, f, 0x1.62bfd47773353p-20);
    g = __builtin_fma(g, f, 0x1.ffcbfc670dcd4p-17);
    g = __builtin_fma(g, f, 0x1.430913096fd9fp-13);
    g = __builtin_fma(g, f, 0x1.5d87fe78a5276p-10);
    g = __builtin_fma(g, f, 0x1.3b2ab6fba1ddap-7);
    g = __builtin_fma(g, f, 0x1.c6b08d704a0c2p-5);
    g = __builtin_fma(g, f, 0x1.ebfbdff82c598p-3);
    g = __builtin_fma(g, f, 0x1.62e42fefa39efp-1);
    return __builtin_fma(g, f, 1.0);
}
__device__ inline double exp64(double x) {
    x = fmax(x, -700.0);
    const double s = __builtin_fma(x, PER_LN2, ONE_AND_A_HALF);
    return add_to_high(exp2_near_0(__builtin_fma(x, PER_LN2, -(s - ONE_AND_A_HALF))), (int)((uint32_t)__double2loint(s) << 20));
}
// The same with the 128 powers 2^(j / 128) in LDS, for one exponential per logit: n counts 128ths, and what is left is so
// small that g takes four nodes (1.5e-16); with the roundings e^x is 4 + |x| units of 2^-53 off at most.  A power lies there
// less its number j in the exponent's lowest bits, so that adding n there gives 2^(n / 128).  Twelve f64 instructions per
// logit, its place in the sum among them; without powers it would be eighteen (64 x 8 rows of 131072 bf16 logits: 77 us instead of 66).
constexpr int POWER_BITS = 7, POWERS = 1 << POWER_BITS;
__device__ inline void fill_powers(double* powers, int t) {
    if (t >= POWERS) return;
    const double power = t <= POWERS / 2 ? exp2_near_0(t * (1.0 / POWERS)) : 2.0 * exp2_near_0(t * (1.0 / POWERS) - 1.0);
    powers[t] = add_to_high(power, -(t << (20 - POWER_BITS)));
}
__device__ inline double exp64(double x, const double* powers) {
    x = fmax(x, -700.0);
    const double s = __builtin_fma(x, POWERS * PER_LN2, ONE_AND_A_HALF);
    const double f = __builtin_fma(x, POWERS * PER_LN2, -(s - ONE_AND_A_HALF));
    const int n = __double2loint(s);
    double g = 0x1.3b2abc07c93d0p-35;
    g = __builtin_fma(g, f, 0x1.c6b0985c8a1bcp-26);
    g = __builtin_fma(g, f, 0x1.ebfbdff82c4edp-17);
    g = __builtin_fma(g, f, 0x1.62e42fefa3892p-8);
    const double power = add_to_high(powers[n & (POWERS - 1)], (int)((uint32_t)n << (20 - POWER_BITS)));
    return __builtin_fma(power, g * f, power);
}

// order-preserving whole number of a double (-0 as +0); 0 for what is never offered (-inf, NaN)
__device__ inline uint64_t order64(double d) {
    if (!(d > -__builtin_inf())) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(d + 0.0);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ inline double of_order64(uint64_t o) {
    return __longlong_as_double((long long)((o >> 63) ? (o & 0x7fffffffffffffffull) : ~o));
}

// ---- across a workgroup ---------------------------------------------------------
__device__ inline uint32_t wave_max(uint32_t v) {
    for (int o = 32; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}
__device__ inline double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// By one wave: the k-th largest of the 64 * PER values of `maxima` (zeros among them count as absent: 0 if there are
// fewer), cut to its upper 20 bits: at least k of the values are >= the result.
template <int PER>
__device__ inline uint32_t kth_largest(const uint32_t* maxima, uint32_t k, uint32_t lane) {
    uint32_t v[PER], t = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = maxima[lane + 64 * i];
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t cand = t | (1u << bit);
        uint32_t cnt = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) cnt += (uint32_t)__popcll(__ballot(v[i] >= cand));
        if (cnt >= k) t = cand;
    }
    return t;
}
// How many of the first n values of `list` lie above each of `mine`; the list is read eight at a time and ends in zeros up
// to the next multiple of eight.
template <int MINE>
__device__ inline void count_above(const uint64_t* list, uint32_t n, const uint64_t (&mine)[MINE], uint32_t (&above)[MINE]) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) above[i] = 0;
    for (uint32_t j = 0; j < n; j += 8) {
        uint64_t o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) o[u] = list[j + u];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int i = 0; i < MINE; ++i) above[i] += o[u] > mine[i];
    }
}
// Sum of one count per thread over the workgroup's WAVES; `slot` is LDS of 2 x WAVES words that two calls in a row use in
// turn.
template <int WAVES>
__device__ inline uint32_t block_count(uint32_t mine, uint32_t* slot, uint32_t turn) {
    for (int o = 32; o; o >>= 1) mine += (uint32_t)__shfl_xor((int)mine, o);
    uint32_t* s = slot + (turn & 1) * WAVES;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = mine;
    __syncthreads();
    uint32_t all = 0;
    for (int w = 0; w < WAVES; ++w) all += s[w];
    return all;
}

struct BeamParams {
    const void* logits;
    const float* scores;      // [rows] or null
    const uint8_t* finished;  // [rows] or null
    const uint32_t* mask;     // or null
    uint64_t row_stride, mask_stride;
    uint32_t rows, groups, beams, vocab, k, end_token;
    uint32_t pieces, chunks_per_piece;  // of a row
    uint32_t len;                           // entries of a piece's list, >= k
    uint32_t per_row_magic, per_row_shift;  // i / (pieces * len) = (i * magic) >> (31 + shift) for i < 2^31
    // per (row, piece)
    uint64_t* list;   // [rows][pieces][len]: order of the logit << 32 | ~token in any order, 0 behind the last
    double* sum;      // [rows][pieces] sum of exp(x - peak)
    float* peak;      // [rows][pieces] largest admitted logit; -inf: none; NaN: a NaN among them
    uint32_t* out_parents;
    uint32_t* out_tokens;
    float* out_scores;
    uint32_t* out_counts;
};

// One piece of one row: chunks_per_piece chunks of PIECE_THREADS * EACH logits, each held in registers while the next one is
// under way.  A list in LDS keeps what can be among the piece's k largest.  What reaches the list has to reach a bound: the
// k-th largest of GROUPS running maxima per thread, which k logits reach; it is found again after 1, 2, 4, 8, ... chunks, so
// that about k log2(chunks) logits are listed in all.  Which logits a thread adds up, and in which order, follows from the
// places and values of its row alone: equal rows have equal sums.
//
// Not normalized it is bound by the bytes: 32 x 10 x 100003 f32, k = 64, take 30 us (4.3 TB/s).
// Normalized the f64 instructions bound it: 64 x 8 x 131072, k = 8, take 66 us in bf16, 74 in f32 (3.6 TB/s).
template <typename V, int EACH, int GROUPS, bool NORMALIZE, bool MASKED>
__global__ __launch_bounds__(PIECE_THREADS) void beam_piece_kernel(BeamParams p) {
    constexpr int WIDE = 16 / V::size, LOADS = EACH / WIDE, CAP = 1024, MINE = CAP / PIECE_THREADS;
    constexpr uint32_t CHUNK = PIECE_THREADS * EACH, LOWEST = 0x00800000u;  // LOWEST: order of the lowest finite f32
    __shared__ uint32_t s_max[PIECE_THREADS * GROUPS];
    __shared__ __align__(16) uint64_t s_list[CAP + 8];
    __shared__ double s_sum[4];
    __shared__ float s_top[4];
    __shared__ double s_powers[NORMALIZE ? POWERS : 1];
    __shared__ uint32_t s_nan, s_add[3], s_bound, s_highest, s_fill;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const uint32_t row = blockIdx.x / p.pieces, piece = blockIdx.x % p.pieces;
    const size_t at = (size_t)row * p.pieces + piece;
    uint64_t* list = p.list + at * p.len;
    const bool ended = p.finished && p.finished[row];
    const float start = p.scores ? p.scores[row] : 0.0f;
    if (ended || !(start > -__builtin_inff())) {  // nothing of this row is looked at
        for (uint32_t i = t; i < p.len; i += PIECE_THREADS)
            list[i] = ended && piece == 0 && i == 0 ? ((uint64_t)f2ord(0.0f) << 32) | (uint32_t)~p.end_token : 0;
        if (t == 0) { p.sum[at] = 0.0; p.peak[at] = -__builtin_inff(); }
        return;
    }
    if (t == 0) { s_nan = 0; s_add[0] = 0; s_add[1] = 0; }
    const typename V::bits* x = (const typename V::bits*)p.logits + (uint64_t)row * p.row_stride;
    const uint32_t* mask = MASKED ? p.mask + (uint64_t)row * p.mask_stride : nullptr;
    const uint32_t first = piece * p.chunks_per_piece * CHUNK;
    const uint32_t behind = (uint32_t)min((uint64_t)p.vocab, (uint64_t)first + (uint64_t)p.chunks_per_piece * CHUNK);

    u32x4 raw[LOADS];
    uint32_t bits[LOADS];
    auto load = [&](uint32_t chunk0) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const uint32_t tok = chunk0 + (j * PIECE_THREADS + t) * WIDE;
            if (tok + WIDE <= p.vocab) {
                raw[j] = *(const u32x4_any*)(x + tok);
            } else {  // -inf behind the end
                typename V::bits one[WIDE];
#pragma unroll
                for (int w = 0; w < WIDE; ++w) one[w] = tok + w < p.vocab ? x[tok + w] : V::round(-__builtin_inff());
                __builtin_memcpy(&raw[j], one, 16);
            }
            if (MASKED) bits[j] = tok < p.vocab ? mask[tok >> 5] >> (tok & 31) : 0;  // WIDE divides 32
        }
    };
    load(first);
    if (NORMALIZE) fill_powers(s_powers, (int)t);  // (the first bound's barriers stand before their use)

    uint32_t n = 0;      // entries of the list
    float bound = 0.0f;  // a logit below it is not among the k largest
    float run[GROUPS];   // largest logits of this thread so far
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) run[g] = -__builtin_inff();
    // The thread's sum of exponentials, in units of exp(ref): ref is the largest logit of the workgroup when the bound was last
    // raised, or a larger one of this thread since.  (In units of the thread's own largest, which grows in most of the first
    // chunks, 64 x 8 rows of 131072 logits take 77 us instead of 74 in f32, 67.5 instead of 66.4 in bf16.)
    double sum = 0.0;
    float ref = -__builtin_inff(), highest = ref;
    bool nan = false;
    uint32_t slot = 0;

    // bound := the k-th largest running maximum; s_highest: the largest
    auto raise = [&] {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) s_max[g * PIECE_THREADS + t] = run[g] > -__builtin_inff() ? f2ord(run[g] + 0.0f) : 0;
        __syncthreads();
        if (wave == 0) {
            const uint32_t kth = kth_largest<4 * GROUPS>(s_max, p.k, lane);
            if (lane == 0) s_bound = max(kth, LOWEST);
        } else if (NORMALIZE && wave == 1) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4 * GROUPS; ++i) m = max(m, s_max[lane + 64 * i]);
            m = wave_max(m);
            if (lane == 0) s_highest = m;
        }
        __syncthreads();
        return ord2f(s_bound);
    };
    // the list cut to its k largest, by counting; true if it held more
    auto cut = [&] {
        if (n <= p.k) return false;
        uint64_t mine[MINE];
        uint32_t rank[MINE];
#pragma unroll
        for (int i = 0; i < MINE; ++i) mine[i] = t + i * PIECE_THREADS < n ? s_list[t + i * PIECE_THREADS] : 0;
        if (t < 8) s_list[n + t] = 0;
        __syncthreads();
        if (n <= PIECE_THREADS) {  // a row's short last piece, mostly: one value per thread
            uint64_t one[1] = {mine[0]};
            uint32_t above[1];
            count_above<1>(s_list, n, one, above);
            rank[0] = above[0];
        } else {
            count_above<MINE>(s_list, n, mine, rank);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MINE; ++i)
            if (mine[i] && rank[i] < p.k) s_list[rank[i]] = mine[i];
        __syncthreads();
        n = p.k;
        return true;
    };

    uint32_t done = 0;
    for (uint32_t chunk0 = first;; chunk0 += CHUNK) {
        float v[EACH];
        bool here = false;  // a NaN in this chunk
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            typename V::bits one[WIDE];
            __builtin_memcpy(one, &raw[j], 16);
#pragma unroll
            for (int w = 0; w < WIDE; ++w) {
                const float f = V::widen(one[w]);
                v[j * WIDE + w] = !MASKED || ((bits[j] >> w) & 1) ? f : -__builtin_inff();
                here |= v[j * WIDE + w] != v[j * WIDE + w];
            }
        }
        if (__any(here)) {
            nan |= here;
#pragma unroll
            for (int e = 0; e < EACH; ++e) v[e] = v[e] != v[e] ? -__builtin_inff() : v[e];
        }
        const bool more = behind - chunk0 > CHUNK;
        if (more) load(chunk0 + CHUNK);
        float top = -__builtin_inff();
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            float m = -__builtin_inff();
#pragma unroll
            for (int e = g * (EACH / GROUPS); e < (g + 1) * (EACH / GROUPS); ++e) m = fmaxf(m, v[e]);
            top = fmaxf(top, m);
            run[g] = fmaxf(run[g], m);
        }
        ++done;
        if ((done & (done - 1)) == 0) {
            const float b = raise();
            bound = done == 1 ? b : fmaxf(bound, b);
            if (NORMALIZE && s_highest) highest = ord2f(s_highest);
        }
        // the logits that reach `least` go behind the list's n entries: one place per wave, then one per logit; how many
        auto append = [&](float least) {
            if (__any(top >= least)) {
                uint32_t cnt = 0;
#pragma unroll
                for (int e = 0; e < EACH; ++e) cnt += (uint32_t)__popcll(__ballot(v[e] >= least));
                uint32_t base = 0;
                if (lane == 0) base = atomicAdd(&s_add[slot], cnt);
                base = n + (uint32_t)__builtin_amdgcn_readfirstlane((int)base);
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const uint64_t who = __ballot(v[e] >= least);
                    if (who) {
                        const uint32_t i = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
                        if (v[e] >= least && i < CAP) {
                            const uint32_t tok = chunk0 + ((e / WIDE) * PIECE_THREADS + t) * WIDE + e % WIDE;
                            s_list[i] = ((uint64_t)f2ord(v[e] + 0.0f) << 32) | (uint32_t)~tok;
                        }
                        base += (uint32_t)__popcll(who);
                    }
                }
            }
            // three counters in turn: the next one was last read before the barrier before this one
            if (t == 0) s_add[slot == 2 ? 0 : slot + 1] = 0;
            __syncthreads();
            const uint32_t add = s_add[slot];
            slot = slot == 2 ? 0 : slot + 1;
            return add;
        };
        uint32_t add = append(bound);
        if (n + add > CAP) {
            // Large logits that come late in the row: this chunk raises the bound itself.  If thousands still reach it
            // (equal ones, or an order that puts all large ones into few threads), one logit of every thread at a time
            // goes to the list, which is cut back as it fills.
            bound = fmaxf(bound, raise());
            add = 0;
            if (n > CAP - PIECE_THREADS && cut()) bound = fmaxf(bound, ord2f((uint32_t)(s_list[n - 1] >> 32)));  // room for one of every thread
            if (t == 0) s_fill = n;
            __syncthreads();
#pragma unroll 1
            for (uint32_t e0 = 0; e0 < EACH; ++e0) {
                float y = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < EACH; ++e) y = e0 == (uint32_t)e ? v[e] : y;
                if (y >= bound) {
                    const uint32_t tok = chunk0 + ((e0 / WIDE) * PIECE_THREADS + t) * WIDE + e0 % WIDE;
                    s_list[atomicAdd(&s_fill, 1u)] = ((uint64_t)f2ord(y + 0.0f) << 32) | (uint32_t)~tok;
                }
                __syncthreads();
                n = s_fill;
                __syncthreads();
                if (n > CAP - PIECE_THREADS && cut()) {
                    bound = fmaxf(bound, ord2f((uint32_t)(s_list[n - 1] >> 32)));
                    if (t == 0) s_fill = n;
                    __syncthreads();
                }
            }
            // the k-th's equals in later chunks come behind it: the next f32
            if (cut()) bound = fmaxf(bound, ord2f((uint32_t)(s_list[n - 1] >> 32) + 1));
        }
        n += add;
        if (NORMALIZE && top > -__builtin_inff()) {
            const float most = fmaxf(top, highest);
            if (most > ref) {  // ref is -inf at first, and the sum 0
                sum *= exp64((double)ref - (double)most, s_powers);
                ref = most;
            }
            const double r = (double)ref;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                sum += exp64((double)v[e] - r, s_powers);
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four at a time: more in flight cost registers, and waves
            }
        }
        if (!more) break;
    }
    if (NORMALIZE) {
        float m = run[0];
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) m = fmaxf(m, run[g]);
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (lane == 0) s_top[wave] = m;
        if (nan) s_nan = 1;
        __syncthreads();
        m = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
        sum = ref > -__builtin_inff() ? sum * exp64((double)ref - (double)m) : 0.0;
        sum = wave_sum(sum);
        if (lane == 0) s_sum[wave] = sum;
        __syncthreads();
        if (t == 0) {
            p.sum[at] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
            p.peak[at] = s_nan ? __uint_as_float(0x7fc00000u) : m;
        }
    }
    if (n > p.len) {  // what the last bound lets through; the k largest by counting if that is still too much
        // (not `bound` itself: after a cut it is past the k-th's value, which stays in the list)
        const uint64_t least = (uint64_t)f2ord(raise()) << 32;
        uint64_t mine[MINE];
#pragma unroll
        for (int i = 0; i < MINE; ++i) mine[i] = t + i * PIECE_THREADS < n ? s_list[t + i * PIECE_THREADS] : 0;
        if (t == 0) s_fill = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MINE; ++i)
            if (mine[i] >= least) s_list[atomicAdd(&s_fill, 1u)] = mine[i];
        __syncthreads();
        n = s_fill;
        if (n > p.len) cut();
    }
    for (uint32_t i = t; i < p.len; i += PIECE_THREADS) list[i] = i < n ? s_list[i] : 0;
}

// One group: the logs of its rows' sums, the totals of what the pieces listed, and the k best of them.  A thread fetches
// AT_ONCE entries at a time.  A chain of short steps by one workgroup: what bounds it are latencies, those of the first
// fetch of each instruction among them, so that less code is faster: 4 beams of 32000 f32 logits take 5.5 us with AT_ONCE 2,
// 6.8 with 8 (and 6.8 with 256 threads and 8); 10240 entries 8.3 with 4, 8.9 with 8.
constexpr uint32_t JOIN_THREADS = 1024, JOIN_AT_ONCE = 4, JOIN_FEW = 2;
template <uint32_t AT_ONCE, int GROUPS, bool NORMALIZE>
__global__ __launch_bounds__(JOIN_THREADS) void beam_join_kernel(BeamParams p) {
    constexpr uint32_t CAP = 2048, JOIN_WAVES = JOIN_THREADS / 64;
    __shared__ double s_lse[BEAMS_MAX];
    __shared__ float s_start[BEAMS_MAX];
    __shared__ uint32_t s_max[256 * GROUPS], s_n, s_bound, s_cnt[2 * JOIN_WAVES];
    __shared__ __align__(16) uint64_t s_ord[CAP + 8];
    __shared__ __align__(16) uint64_t s_entry[CAP];
    __shared__ __align__(16) uint16_t s_beam[CAP];
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, group = blockIdx.x;
    const size_t row0 = (size_t)group * p.beams;
    const uint64_t* list = p.list + row0 * p.pieces * p.len;
    const uint32_t slots = p.beams * p.pieces * p.len;  // below 2^31
    auto fetch = [&](uint32_t i0, uint64_t (&e)[AT_ONCE]) {
#pragma unroll
        for (uint32_t u = 0; u < AT_ONCE; ++u) e[u] = i0 + u * JOIN_THREADS < slots ? list[i0 + u * JOIN_THREADS] : 0;
    };
    uint64_t head[AT_ONCE];  // the first entries: under way while the logs are taken, and kept
    fetch(t, head);
    // As many lanes to a row as it has pieces (up to 64, a power of two): 1000 beams of one piece each took 100 us with a
    // wave per row.
    uint32_t lanes = 1;
    while (lanes < 64 && lanes < p.pieces) lanes *= 2;
    const uint32_t sub = lane & (lanes - 1);
    for (uint32_t b = t / lanes; b < p.beams; b += JOIN_THREADS / lanes) {
        const size_t at = (row0 + b) * p.pieces;
        const float start = p.scores ? p.scores[row0 + b] : 0.0f;
        double lse = 0.0;
        if (NORMALIZE && !(p.finished && p.finished[row0 + b])) {
            float m = -__builtin_inff();
            uint32_t bad = 0;
            double s = 0.0;
            for (uint32_t i0 = 0; i0 < p.pieces; i0 += lanes) {  // (a row of more than 64 pieces: its sums are scaled as its maximum grows)
                const bool in = i0 + sub < p.pieces;
                const float v = in ? p.peak[at + i0 + sub] : -__builtin_inff();
                const double part = in ? p.sum[at + i0 + sub] : 0.0;
                bad |= v != v;
                float most = fmaxf(m, v);
                for (uint32_t o = lanes / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, (int)o));
                if (most > -__builtin_inff()) s = (m > -__builtin_inff() ? s * exp64((double)m - (double)most) : 0.0) + (v > -__builtin_inff() ? part * exp64((double)v - (double)most) : 0.0);
                m = most;
            }
            for (uint32_t o = lanes / 2; o; o >>= 1) {
                bad |= (uint32_t)__shfl_xor((int)bad, (int)o);
                s += __shfl_xor(s, (int)o);
            }
            lse = bad || m == __builtin_inff() ? __longlong_as_double(0x7ff8000000000000ll) : (double)m + log(s);
        }
        if (sub == 0) {
            s_lse[b] = lse;
            s_start[b] = start;
        }
    }
    if (t == 0) s_n = 0;
    for (uint32_t i = t; i < 256 * GROUPS; i += JOIN_THREADS) s_max[i] = 0;
    __syncthreads();
    // order of the total and beam of a list entry; an ended beam's entry holds a logit of 0 and no sum
    auto total_of = [&](uint64_t e, uint32_t i, uint32_t* beam) -> uint64_t {
        const uint32_t b = (uint32_t)(((uint64_t)i * p.per_row_magic) >> (31 + p.per_row_shift));
        *beam = b;
        return e ? order64((double)s_start[b] + ((double)ord2f((uint32_t)(e >> 32)) - s_lse[b])) : 0;
    };
    // f(order, entry, beam, slot) for every slot that holds an entry of a total
    auto each = [&](auto f) {
        for (uint32_t i0 = t; i0 < slots; i0 += JOIN_THREADS * AT_ONCE) {
            uint64_t e[AT_ONCE];
            if (i0 != t) fetch(i0, e);
#pragma unroll
            for (uint32_t u = 0; u < AT_ONCE; ++u) {
                const uint64_t entry = i0 == t ? head[u] : e[u];
                uint32_t beam = 0;
                const uint64_t o = entry ? total_of(entry, i0 + u * JOIN_THREADS, &beam) : 0;
                if (o) f(o, entry, beam, i0 + u * JOIN_THREADS);
            }
        }
    };
    // Maxima over 256 * GROUPS sets of entries; a piece's entries stand at the front of its list, so the sets are mixed by a
    // hash of the slot: large totals that shared a set would lower the bound.
    each([&](uint64_t o, uint64_t, uint32_t, uint32_t i) {
        atomicMax(&s_max[(i * 2654435761u) >> (GROUPS == 1 ? 24 : 22)], (uint32_t)(o >> 32));
    });
    __syncthreads();
    if (wave == 0) {
        const uint32_t kth = kth_largest<4 * GROUPS>(s_max, p.k, lane);
        if (lane == 0) s_bound = kth;
    }
    __syncthreads();
    const uint32_t bound = s_bound;
    auto keep = [&](uint64_t o, uint64_t e, uint32_t beam) {
        const uint32_t at = atomicAdd(&s_n, 1u);
        if (at < CAP) { s_ord[at] = o; s_entry[at] = e; s_beam[at] = (uint16_t)beam; }
    };
    each([&](uint64_t o, uint64_t e, uint32_t beam, uint32_t) {
        if ((uint32_t)(o >> 32) >= bound) keep(o, e, beam);
    });
    __syncthreads();
    uint32_t n = s_n;
    if (n > CAP) {
        // thousands of totals a 2^-20th apart: the exact k-th of them bit by bit -- its total, its beam among those that
        // equal it, its entry among that beam's
        uint32_t turn = 0, last_beam = 0, c;
        uint64_t kth = 0, last = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t cand = kth | (1ull << bit);
            c = 0;
            each([&](uint64_t o, uint64_t, uint32_t, uint32_t) { c += o >= cand; });
            if (block_count<JOIN_WAVES>(c, s_cnt, turn++) >= p.k) kth = cand;
        }
        c = 0;
        each([&](uint64_t o, uint64_t, uint32_t, uint32_t) { c += o > kth; });
        uint32_t need = p.k - block_count<JOIN_WAVES>(c, s_cnt, turn++);
        for (int bit = 9; bit >= 0; --bit) {  // the largest beam that fewer than `need` of the equal ones lie before
            const uint32_t cand = last_beam | (1u << bit);
            c = 0;
            each([&](uint64_t o, uint64_t, uint32_t b, uint32_t) { c += o == kth && b < cand; });
            if (block_count<JOIN_WAVES>(c, s_cnt, turn++) < need) last_beam = cand;
        }
        c = 0;
        each([&](uint64_t o, uint64_t, uint32_t b, uint32_t) { c += o == kth && b < last_beam; });
        need -= block_count<JOIN_WAVES>(c, s_cnt, turn++);
        for (int bit = 63; bit >= 0; --bit) {  // entries count down: ~entry ascends
            const uint64_t cand = last | (1ull << bit);
            c = 0;
            each([&](uint64_t o, uint64_t e, uint32_t b, uint32_t) { c += o == kth && b == last_beam && ~e < cand; });
            if (block_count<JOIN_WAVES>(c, s_cnt, turn++) < need) last = cand;
        }
        __syncthreads();
        if (t == 0) s_n = 0;
        __syncthreads();
        each([&](uint64_t o, uint64_t e, uint32_t b, uint32_t) {
            if (o > kth || (o == kth && (b < last_beam || (b == last_beam && ~e <= last)))) keep(o, e, b);
        });
        __syncthreads();
        n = s_n;  // k
    }
    uint32_t* parents = p.out_parents + (size_t)group * p.k;
    uint32_t* tokens = p.out_tokens + (size_t)group * p.k;
    float* scores = p.out_scores + (size_t)group * p.k;
    if (t < 8) s_ord[n + t] = 0;
    __syncthreads();
    // Ranks by counting, as many threads to an entry as there are (up to 16).  Equal totals -- half-precision logits of one
    // beam are often equal -- are told apart by beam, then by logit and token.
    uint32_t share = 1;
    while (share < 16 && n * share * 2 <= JOIN_THREADS) share *= 2;
    for (uint32_t i0 = 0; i0 < n; i0 += JOIN_THREADS / share) {
        const uint32_t i = i0 + t / share;
        uint32_t rank = 0, b = 0;
        uint64_t o = 0, e = 0;
        if (i < n) {
            o = s_ord[i];
            e = s_entry[i];
            b = s_beam[i];
            for (uint32_t j = t % share * 8; j < n; j += share * 8) {
                uint64_t other[8];
                bool same = false;
#pragma unroll
                for (int u = 0; u < 8; ++u) other[u] = s_ord[j + u];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    rank += other[u] > o;
                    same |= other[u] == o && j + u != i;
                }
                if (same) {
                    uint64_t entry[8];
                    uint16_t beam[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) { entry[u] = s_entry[j + u]; beam[u] = s_beam[j + u]; }
#pragma unroll
                    for (int u = 0; u < 8; ++u) rank += other[u] == o && (beam[u] < b || (beam[u] == b && entry[u] > e));
                }
            }
        }
        for (uint32_t q = 1; q < share; q *= 2) rank += (uint32_t)__shfl_xor((int)rank, (int)q);
        if (i < n && rank < p.k && t % share == 0) {
            parents[rank] = b;
            tokens[rank] = (uint32_t)~(uint32_t)e;
            scores[rank] = (float)of_order64(o);
        }
    }
    for (uint32_t i = n + t; i < p.k; i += JOIN_THREADS) {
        parents[i] = tokens[i] = 0xffffffffu;
        scores[i] = -__builtin_inff();
    }
    if (t == 0) p.out_counts[group] = min(n, p.k);
}

// ---- the move of the states -------------------------------------------------------------------
constexpr uint32_t STATES_PER_LAUNCH = 8, STATES_MAX = 256;
constexpr uint32_t MOVE_BYTES = 4096;  // of one run, by one wave at a time
struct MoveParams {
    needle_beam_state s[STATES_PER_LAUNCH];
    uint64_t first[STATES_PER_LAUNCH + 1];  // moves before state i; a move is MOVE_BYTES of a run
    const uint32_t* parents;
    uint32_t n_states, groups, beams, k;
};

__global__ __launch_bounds__(256) void beam_move_kernel(MoveParams p) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t step = (uint64_t)gridDim.x * 4, rows = (uint64_t)p.groups * p.k;
    for (uint64_t m = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); m < p.first[p.n_states]; m += step) {
        uint32_t i = 0;
        while (m >= p.first[i + 1]) ++i;
        const needle_beam_state& s = p.s[i];
        uint64_t at = m - p.first[i];
        const uint64_t cuts = (s.bytes + MOVE_BYTES - 1) / MOVE_BYTES;
        const uint64_t cut = at % cuts;
        at /= cuts;
        const uint64_t in = at % s.inner;
        at /= s.inner;
        const uint64_t row = at % rows, out = at / rows;
        const uint32_t parent = p.parents[row];
        if (parent >= p.beams) continue;
        const uint64_t from = row / p.k * p.beams + parent;
        const uint8_t* src = (const uint8_t*)s.src + out * s.src_outer_stride + from * s.src_row_stride + in * s.src_inner_stride + cut * MOVE_BYTES;
        uint8_t* dst = (uint8_t*)s.dst + out * s.dst_outer_stride + row * s.dst_row_stride + in * s.dst_inner_stride + cut * MOVE_BYTES;
        const uint32_t len = (uint32_t)min((uint64_t)MOVE_BYTES, s.bytes - cut * MOVE_BYTES);
        u32x4 v[MOVE_BYTES / 1024];
#pragma unroll
        for (uint32_t j = 0; j < MOVE_BYTES / 1024; ++j)
            if (j * 1024 + lane * 16 + 16 <= len) v[j] = *(const u32x4_any*)(src + j * 1024 + lane * 16);
#pragma unroll
        for (uint32_t j = 0; j < MOVE_BYTES / 1024; ++j)
            if (j * 1024 + lane * 16 + 16 <= len) *(u32x4_any*)(dst + j * 1024 + lane * 16) = v[j];
        const uint32_t whole = len & ~15u;
        if (lane < len - whole) dst[whole + lane] = src[whole + lane];
    }
}

static hipError_t launch_moves(const uint32_t* d_parents, uint32_t groups, uint32_t beams, uint32_t k, const needle_beam_state* states,
                               uint32_t n_states, int n_cu, hipStream_t stream) {
    MoveParams p{};
    p.parents = d_parents; p.groups = groups; p.beams = beams; p.k = k;
    for (uint32_t i = 0; i < n_states; ++i) {
        const needle_beam_state& s = states[i];
        const uint64_t moves = s.outer * s.inner * groups * k * ((s.bytes + MOVE_BYTES - 1) / MOVE_BYTES);
        if (moves) {
            p.s[p.n_states] = s;
            p.first[p.n_states + 1] = p.first[p.n_states] + moves;
            ++p.n_states;
        }
        if (p.n_states == STATES_PER_LAUNCH || (i + 1 == n_states && p.n_states)) {
            const uint64_t blocks = std::min<uint64_t>((p.first[p.n_states] + 3) / 4, (uint64_t)n_cu * 16);
            hipLaunchKernelGGL(beam_move_kernel, dim3((uint32_t)blocks), dim3(256), 0, stream, p);
            p.n_states = 0;
        }
    }
    return hipGetLastError();
}

// ---- host side ---------------------------------------------------------------------------------
// Bytes of a row per thread and chunk.  Us with 32 and with 64: 64 x 8 rows of 131072 logits in bf16 66 and 65, in f32 74 and
// 70; 10 rows of 131000 in bf16, k = 64, 14.2 and 15.0; 4 rows of 32000 in f32 5.8 and 7.3.
constexpr uint32_t CHUNK_BYTES = 32;
// Workgroups per CU that the pieces are cut for: the bf16 rows of 131072 take 66 us with 4, 72 with 5, 69 with 8; 32 x 10 rows of
// 100003 f32 logits, not normalized, 30, 30 and 33.
constexpr uint32_t PIECES_PER_CU = 4;
// What a chunk takes a piece: 1 to 3 us, more with the logarithm and with a larger k.  10 rows of 131000 bf16 logits, k = 64,
// take 23 us with pieces cut for it and 34 with a piece per chunk; 4 rows of 1500000 34, and 42 where it is a tenth.
constexpr double CHUNK_NS = 2000.0;
constexpr uint32_t JOIN_ENTRIES = 8192;
template <typename V, int EACH, int GROUPS>
static void launch_pieces_of(const BeamParams& p, bool normalize, hipStream_t stream) {
    const dim3 grid(p.rows * p.pieces), block(PIECE_THREADS);
    if (normalize && p.mask) hipLaunchKernelGGL((beam_piece_kernel<V, EACH, GROUPS, true, true>), grid, block, 0, stream, p);
    else if (normalize) hipLaunchKernelGGL((beam_piece_kernel<V, EACH, GROUPS, true, false>), grid, block, 0, stream, p);
    else if (p.mask) hipLaunchKernelGGL((beam_piece_kernel<V, EACH, GROUPS, false, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((beam_piece_kernel<V, EACH, GROUPS, false, false>), grid, block, 0, stream, p);
}
template <typename V>
static void launch_pieces(const BeamParams& p, bool normalize, hipStream_t stream) {
    // 256 maxima tell the k <= 64 largest of a chunk well enough (about 1.2 k logits reach the bound), more need 1024
    if (p.k <= 64) launch_pieces_of<V, (int)CHUNK_BYTES / V::size, 1>(p, normalize, stream);
    else launch_pieces_of<V, (int)CHUNK_BYTES / V::size, 4>(p, normalize, stream);
}

template <uint32_t AT_ONCE, int GROUPS>
static void launch_join_of(const BeamParams& p, bool normalize, hipStream_t stream) {
    if (normalize) hipLaunchKernelGGL((beam_join_kernel<AT_ONCE, GROUPS, true>), dim3(p.groups), dim3(JOIN_THREADS), 0, stream, p);
    else hipLaunchKernelGGL((beam_join_kernel<AT_ONCE, GROUPS, false>), dim3(p.groups), dim3(JOIN_THREADS), 0, stream, p);
}
static void launch_join(const BeamParams& p, bool normalize, hipStream_t stream) {
    if (p.k > 64) launch_join_of<JOIN_AT_ONCE, 4>(p, normalize, stream);
    else if (p.beams * p.pieces * p.len > JOIN_FEW * JOIN_THREADS) launch_join_of<JOIN_AT_ONCE, 1>(p, normalize, stream);
    else launch_join_of<JOIN_FEW, 1>(p, normalize, stream);
}

struct ByteRange { const void* p; uint64_t n; };
// Runs of `bytes` bytes from `base` on along three axes; `span` bytes from the first to behind the last.
struct Axis { uint64_t n, stride; };
struct Runs {
    uint64_t base, bytes, span;
    Axis ax[3];
    // one period of them, `at` bytes from its start: without the axes that step by whole periods
    Runs within(uint64_t period, uint64_t at) const {
        Runs r{at, bytes, bytes, {}};
        for (int i = 0; i < 3; ++i)
            if (ax[i].n > 1 && ax[i].stride % period) {
                r.ax[i] = ax[i];
                r.span += (ax[i].n - 1) * ax[i].stride;
            }
        return r;
    }
};
// Two arrays of runs share no byte: one lies behind the other, or they share none of a period that one of their strides
// makes and that neither's runs leave (parts of the rows, the layers or the runs of one array).  Every period leaves out
// an axis, so this ends.
static bool share_nothing(const Runs& a, const Runs& b) {
    if (!a.span || !b.span || a.base + a.span <= b.base || b.base + b.span <= a.base) return true;
    for (const Runs* r : {&a, &b})
        for (const Axis& x : r->ax) {
            if (x.n <= 1 || !x.stride) continue;
            const uint64_t far = a.base < b.base ? (b.base - a.base) % x.stride : (a.base - b.base) % x.stride;
            for (const uint64_t at : {far, (x.stride - far) % x.stride}) {  // (the first run of either may start the period)
                const bool later = (a.base < b.base) == (at == far);  // b's does not
                const Runs first = (later ? a : b).within(x.stride, 0), second = (later ? b : a).within(x.stride, at);
                if (first.span <= x.stride && second.span <= x.stride - at && share_nothing(first, second)) return true;
            }
        }
    return false;
}
// `others`: arrays of the same call that no dst may overlap
static needle_hip_status states_check(const needle_beam_state* states, uint32_t n_states, uint64_t rows, uint64_t picks, const ByteRange* others,
                                      int n_others) {
    if (n_states && !states) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "states is null");
    if (n_states > STATES_MAX) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "at most %u states per call", STATES_MAX);
    Runs from[STATES_MAX], to[STATES_MAX];  // set as far as there are states
    for (uint32_t i = 0; i < n_states; ++i) {
        const needle_beam_state& s = states[i];
        from[i].span = to[i].span = 0;
        if (s.outer == 0 || s.inner == 0 || s.bytes == 0) continue;
        if (!s.src || !s.dst) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "state %u has a null pointer", i);
        // rows, outer and inner runs of dst lie apart in one of their orders: no byte is written twice
        Axis ax[3] = {{s.outer, s.dst_outer_stride}, {picks, s.dst_row_stride}, {s.inner, s.dst_inner_stride}};
        std::sort(ax, ax + 3, [](const Axis& a, const Axis& b) { return a.n > 1 && b.n > 1 ? a.stride < b.stride : a.n > b.n; });
        uint64_t span = s.bytes, last;
        for (const Axis& a : ax) {
            if (a.n <= 1) continue;
            if (a.stride < span) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "rows of state %u overlap in dst", i);
            if (__builtin_mul_overflow(a.n - 1, a.stride, &last) || __builtin_add_overflow(span, last, &span) || span > (1ull << 62))
                return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "state %u spans more than 2^62 bytes", i);
        }
        uint64_t reach = s.bytes;
        const Axis sx[3] = {{s.outer, s.src_outer_stride}, {rows, s.src_row_stride}, {s.inner, s.src_inner_stride}};
        for (const Axis& a : sx)
            if (a.n == 0 || __builtin_mul_overflow(a.n - 1, a.stride, &last) || __builtin_add_overflow(reach, last, &reach) || reach > (1ull << 62))
                return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "state %u spans more than 2^62 bytes", i);
        from[i] = {(uint64_t)s.src, s.bytes, reach, {sx[0], sx[1], sx[2]}};
        to[i] = {(uint64_t)s.dst, s.bytes, span, {ax[0], ax[1], ax[2]}};
        for (int o = 0; o < n_others; ++o)
            if (ranges_meet(s.dst, span, others[o].p, others[o].n))
                return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "dst of state %u overlaps another array of the call", i);
    }
    for (uint32_t i = 0; i < n_states; ++i)
        for (uint32_t j = 0; j < n_states; ++j) {
            if (!share_nothing(to[i], from[j]))
                return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "dst of state %u overlaps src of state %u", i, j);
            if (i < j && !share_nothing(to[i], to[j]))
                return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "dst of state %u overlaps dst of state %u", i, j);
        }
    return NEEDLE_HIP_OK;
}

static needle_hip_status shape_check(uint32_t groups, uint32_t beams, uint32_t k) {
    if (k > BEAM_K_MAX) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "k = %u exceeds %u", k, BEAM_K_MAX);
    if (beams > BEAMS_MAX) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "beams = %u exceeds %u", beams, BEAMS_MAX);
    if ((uint64_t)groups * beams >= (1ull << 31) || (uint64_t)groups * k >= (1ull << 31))
        return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "at most 2^31-1 beams and picks per call");
    return NEEDLE_HIP_OK;
}

static needle_hip_status select_check(needle_hip_ctx* c, const needle_beam_params* q, const void* logits, const needle_beam_state* states,
                                      uint32_t n_states, const uint32_t* parents, const uint32_t* tokens, const float* scores,
                                      const uint32_t* counts) {
    if (!c || !q) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "null argument");
    if (!value_known(q->value)) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "unknown value type %d", q->value);
    if (q->reserved) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "reserved is not 0");
    ST_TRY(shape_check(q->groups, q->beams, q->k));
    if (q->vocab >= (1u << 31)) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "vocab reaches 2^31");
    if ((uint64_t)q->beams * q->vocab >= (1ull << 32)) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "beams * vocab reaches 2^32");
    if (q->groups == 0) return NEEDLE_HIP_OK;
    if (!counts || (q->k && (!parents || !tokens || !scores))) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "null output pointer");
    const uint64_t rows = (uint64_t)q->groups * q->beams;
    if (rows == 0 || q->k == 0) return NEEDLE_HIP_OK;
    if (q->vocab && !logits) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "logits is null");
    if (q->finished && q->end_token >= q->vocab) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "end_token %u is not below vocab %u", q->end_token, q->vocab);
    if (rows > 1 && q->row_stride < q->vocab) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "row_stride is smaller than vocab");
    const uint64_t words = ((uint64_t)q->vocab + 31) / 32;
    if (q->mask && q->mask_stride && q->mask_stride < words) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "mask_stride is smaller than a row's mask");
    if ((uintptr_t)logits % value_size(q->value) || ((uintptr_t)q->scores | (uintptr_t)q->mask | (uintptr_t)parents | (uintptr_t)tokens | (uintptr_t)scores | (uintptr_t)counts) % 4)
        return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its element");
    uint64_t nl, nm;
    if (!span_bytes(rows, q->vocab, q->row_stride, value_size(q->value), &nl) || !span_bytes(q->mask_stride ? rows : 1, words, q->mask_stride, 4, &nm))
        return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "an array spans more than 2^62 bytes");
    const uint64_t np = (uint64_t)q->groups * q->k * 4;
    const ByteRange outs[4] = {{parents, np}, {tokens, np}, {scores, np}, {counts, (uint64_t)q->groups * 4}},
                    ins[4] = {{logits, nl}, {q->scores, rows * 4}, {q->finished, rows}, {q->mask, nm}};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (ranges_meet(outs[i].p, outs[i].n, ins[j].p, ins[j].n) || (i != j && ranges_meet(outs[i].p, outs[i].n, outs[j].p, outs[j].n)))
                return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "an output overlaps another array");
    if (n_states) {
        const ByteRange all[8] = {outs[0], outs[1], outs[2], outs[3], ins[0], ins[1], ins[2], ins[3]};
        ST_TRY(states_check(states, n_states, rows, (uint64_t)q->groups * q->k, all, 8));
    }
    return NEEDLE_HIP_OK;
}

__global__ void beam_empty_kernel(uint32_t* parents, uint32_t* tokens, float* scores, uint32_t* counts, uint32_t groups, uint32_t k) {
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (uint64_t)groups * max(k, 1u); i += (uint64_t)gridDim.x * blockDim.x) {
        if (k) { parents[i] = tokens[i] = 0xffffffffu; scores[i] = -__builtin_inff(); }
        if (i < groups) counts[i] = 0;
    }
}

// enqueues the selection on the context's stream; the caller holds the context's lock
static needle_hip_status select_enqueue(needle_hip_ctx* c, const needle_beam_params& q, const void* d_logits, uint32_t* parents,
                                        uint32_t* tokens, float* scores, uint32_t* counts) {
    if (q.k == 0 || q.beams == 0 || q.vocab == 0) {
        hipLaunchKernelGGL(beam_empty_kernel, dim3(std::min<uint32_t>((uint32_t)(((uint64_t)q.groups * std::max(q.k, 1u) + 255) / 256), 4096)), dim3(256), 0,
                           c->stream, parents, tokens, scores, counts, q.groups, q.k);
        HIP_TRY(hipGetLastError());
        return NEEDLE_HIP_OK;
    }
    const bool normalize = q.normalize != 0;
    BeamParams p{};
    p.beams = q.beams; p.vocab = q.vocab; p.k = q.k; p.end_token = q.end_token;
    p.row_stride = q.row_stride; p.mask_stride = q.mask_stride;
    p.len = std::max<uint32_t>(q.k + q.k / 2, 16);  // room for what the last bound lets through, so that few lists need an exact cut
    // As many pieces as give the chip PIECES_PER_CU workgroups per CU; but a group's lists meet in one workgroup, which takes
    // 3 us longer for JOIN_ENTRIES of them than for a few and then 0.5 ns per entry, while a chunk takes a piece CHUNK_NS:
    // the count where the two add up to least.
    const uint64_t all_rows = (uint64_t)q.groups * q.beams, chunk = PIECE_THREADS * CHUNK_BYTES / value_size(q.value), chunks = (q.vocab + chunk - 1) / chunk;
    const uint64_t share = ((uint64_t)PIECES_PER_CU * c->n_cu + all_rows - 1) / all_rows, entries = (uint64_t)q.beams * p.len;
    const uint64_t joined = std::max<uint64_t>(JOIN_ENTRIES / entries, (uint64_t)std::sqrt((double)chunks * CHUNK_NS / (0.5 * (double)entries)));
    const uint64_t want = std::max<uint64_t>(1, std::min(chunks, std::min(share, joined)));
    p.chunks_per_piece = (uint32_t)((chunks + want - 1) / want);
    p.pieces = (uint32_t)((chunks + p.chunks_per_piece - 1) / p.chunks_per_piece);
    {
        const uint32_t d = p.pieces * p.len;  // rounded up 32-bit reciprocal: exact for numerators below 2^31
        while ((1ull << p.per_row_shift) < d) ++p.per_row_shift;
        p.per_row_magic = (uint32_t)((((1ull << 31) << p.per_row_shift) + d - 1) / d);
    }
    // a block of groups at a time: the pieces' lists stay within 256 MiB (one group's may be more), the grid within 2^22
    const uint64_t group_pieces = (uint64_t)q.beams * p.pieces, piece_bytes = (uint64_t)p.len * 8 + 12;
    uint64_t blk = std::min<uint64_t>((256ull << 20) / (group_pieces * piece_bytes), (1u << 22) / group_pieces);
    blk = std::max<uint64_t>(1, std::min<uint64_t>(blk, q.groups));
    HIP_TRY(c->scratch[7].ensure(blk * group_pieces * piece_bytes));
    p.list = c->scratch[7].as<uint64_t>();
    p.sum = (double*)(p.list + blk * group_pieces * p.len);
    p.peak = (float*)(p.sum + blk * group_pieces);
    for (uint64_t g0 = 0; g0 < q.groups; g0 += blk) {
        const uint64_t r0 = g0 * q.beams;
        p.groups = (uint32_t)std::min<uint64_t>(blk, q.groups - g0);
        p.rows = p.groups * q.beams;
        p.logits = (const unsigned char*)d_logits + r0 * q.row_stride * value_size(q.value);
        p.scores = q.scores ? q.scores + r0 : nullptr;
        p.finished = q.finished ? q.finished + r0 : nullptr;
        p.mask = q.mask ? q.mask + r0 * q.mask_stride : nullptr;
        p.out_parents = parents + g0 * q.k; p.out_tokens = tokens + g0 * q.k; p.out_scores = scores + g0 * q.k; p.out_counts = counts + g0;
        switch (q.value) {
        case NEEDLE_VALUE_F32: launch_pieces<ValueF32>(p, normalize, c->stream); break;
        case NEEDLE_VALUE_F16: launch_pieces<ValueF16>(p, normalize, c->stream); break;
        default: launch_pieces<ValueBF16>(p, normalize, c->stream);
        }
        HIP_TRY(hipGetLastError());
        launch_join(p, normalize, c->stream);
        HIP_TRY(hipGetLastError());
    }
    return NEEDLE_HIP_OK;
}

}  // namespace nh

using namespace nh;

extern "C" needle_hip_status needle_hip_beam_select_device(needle_hip_ctx* c, const needle_beam_params* q, const void* d_logits,
                                                           const needle_beam_state* states, uint32_t n_states, uint32_t* d_out_parents,
                                                           uint32_t* d_out_tokens, float* d_out_scores, uint32_t* d_out_counts) {
    ST_TRY(select_check(c, q, d_logits, states, n_states, d_out_parents, d_out_tokens, d_out_scores, d_out_counts));
    if (q->groups == 0) return NEEDLE_HIP_OK;
    const bool moves = n_states && q->k && q->beams;
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    ST_TRY(select_enqueue(c, *q, d_logits, d_out_parents, d_out_tokens, d_out_scores, d_out_counts));
    if (moves) HIP_TRY(launch_moves(d_out_parents, q->groups, q->beams, q->k, states, n_states, c->n_cu, c->stream));
    HIP_TRY(wait_done(c));
    return NEEDLE_HIP_OK;
}

extern "C" needle_hip_status needle_hip_beam_select(needle_hip_ctx* c, const needle_beam_params* q, const void* logits,
                                                    uint32_t* out_parents, uint32_t* out_tokens, float* out_scores, uint32_t* out_counts) {
    if (!c || !q) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "null argument");
    needle_beam_params h = *q;
    h.row_stride = h.vocab;
    const uint64_t words = ((uint64_t)h.vocab + 31) / 32;
    ST_TRY(select_check(c, &h, logits, nullptr, 0, out_parents, out_tokens, out_scores, out_counts));
    if (h.mask && h.mask_stride && h.mask_stride != words) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "mask_stride is neither 0 nor a row's mask");
    if (h.groups == 0) return NEEDLE_HIP_OK;
    const size_t rows = (size_t)h.groups * h.beams, picks = (size_t)h.groups * h.k;
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    const void* src[4] = {logits, h.scores, h.finished, h.mask};
    const size_t sizes[8] = {rows * h.vocab * value_size(h.value), h.scores ? rows * 4 : 0, h.finished ? rows : 0,
                             h.mask ? (h.mask_stride ? rows : 1) * words * 4 : 0, picks * 4, picks * 4, picks * 4, (size_t)h.groups * 4};
    size_t at[9] = {0};
    for (int i = 0; i < 8; ++i) at[i + 1] = at[i] + ((sizes[i] + 15) & ~(size_t)15);
    HIP_TRY(c->scratch[2].ensure(at[8]));
    unsigned char* d = c->scratch[2].as<unsigned char>();
    if (h.k && h.beams)
        for (int i = 0; i < 4; ++i)
            if (src[i] && sizes[i]) HIP_TRY(hipMemcpyAsync(d + at[i], src[i], sizes[i], hipMemcpyHostToDevice, c->stream));
    h.scores = h.scores ? (const float*)(d + at[1]) : nullptr;
    h.finished = h.finished ? d + at[2] : nullptr;
    h.mask = h.mask ? (const uint32_t*)(d + at[3]) : nullptr;
    ST_TRY(select_enqueue(c, h, d, (uint32_t*)(d + at[4]), (uint32_t*)(d + at[5]), (float*)(d + at[6]), (uint32_t*)(d + at[7])));
    void* dst[4] = {out_parents, out_tokens, out_scores, out_counts};
    for (int i = 0; i < 4; ++i)
        if (sizes[4 + i]) HIP_TRY(hipMemcpyAsync(dst[i], d + at[4 + i], sizes[4 + i], hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}

extern "C" needle_hip_status needle_hip_beam_reorder_device(needle_hip_ctx* c, const uint32_t* d_parents, uint32_t groups, uint32_t beams,
                                                            uint32_t k, const needle_beam_state* states, uint32_t n_states) {
    if (!c) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "ctx is null");
    if (n_states && !states) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "states is null");
    if ((uint64_t)groups * beams >= (1ull << 31) || (uint64_t)groups * k >= (1ull << 31))
        return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "at most 2^31-1 beams and picks per call");
    if (groups == 0 || beams == 0 || k == 0 || n_states == 0) return NEEDLE_HIP_OK;
    if (!d_parents) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "parents is null");
    const ByteRange picks{d_parents, (uint64_t)groups * k * 4};
    ST_TRY(states_check(states, n_states, (uint64_t)groups * beams, (uint64_t)groups * k, &picks, 1));
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    HIP_TRY(launch_moves(d_parents, groups, beams, k, states, n_states, c->n_cu, c->stream));
    HIP_TRY(wait_done(c));
    return NEEDLE_HIP_OK;
}
