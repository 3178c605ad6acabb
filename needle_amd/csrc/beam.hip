// One step of a beam search: the k best continuations over the beams of every group, and the move of what the beams
// carry to their picks' places.
//
//   total(b, t) = scores[b] + x[b][t] - lse[b],   lse[b] = log sum_t exp x[b][t] over the admitted t (0 without normalize)
//
// lse is one number per row, so within a row the order of the totals is the order of the logits: one pass over the logits
// keeps, per piece of a row, its maximum, its sum of exponentials and its k largest logits; a second, small kernel joins the
// pieces of a group.  The pass is bound by the bytes of the logits.
//
// Picks are whole numbers and two beams' totals may lie a rounding apart, so whatever decides between beams is held in
// 64 bits: the exponentials, their sums, the totals.  (f64 fused multiply-adds issue at the rate of f32 ones here.)
#include "nh_values.h"

namespace nh {

constexpr uint32_t BEAM_K_MAX = 256, BEAMS_MAX = 1024;
constexpr uint32_t PIECE_THREADS = 256;

// ---- exponential of x <= 0 in 64 bits -------------------------------------------------------
// exp x = 2^n exp f with n = rint(x / ln 2), |f| <= ln 2 / 2, and exp f by its Taylor series to f^9: the first term left
// out is below 2^-37 * 2^-1.5 / 10! ~ 7e-12 of the result.  Below -800 the result is 0 (as exp's own, from -746 on).
__device__ inline double exp_below0(double x) {
    x = fmax(x, -800.0);
    const double n = rint(x * 1.4426950408889634074);
    const double f = __builtin_fma(n, -0.69314718055994530942, x);
    double p = 2.7557319223985893e-06;  // 1 / 9!
    p = __builtin_fma(p, f, 2.4801587301587302e-05);
    p = __builtin_fma(p, f, 1.9841269841269841e-04);
    p = __builtin_fma(p, f, 1.3888888888888889e-03);
    p = __builtin_fma(p, f, 8.3333333333333333e-03);
    p = __builtin_fma(p, f, 4.1666666666666667e-02);
    p = __builtin_fma(p, f, 1.6666666666666667e-01);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    return ldexp(p, (int)n);
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

// ---- across a workgroup of 4 waves ---------------------------------------------------------
__device__ inline uint32_t wave_max(uint32_t v) {
    for (int o = 32; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}
__device__ inline double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// The k-th largest of the 64 * PER values of `maxima` (zeros among them count as absent: 0 if there are fewer), cut to
// its upper 20 bits: at least k of the values are >= the result.  Every wave computes it for itself.
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
// Sum of one count per thread over the workgroup; `slot` is LDS of 2 x 4 words that two calls in a row use in turn.
__device__ inline uint32_t block_count(uint32_t mine, uint32_t* slot, uint32_t turn) {
    for (int o = 32; o; o >>= 1) mine += (uint32_t)__shfl_xor((int)mine, o);
    uint32_t* s = slot + (turn & 1) * 4;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = mine;
    __syncthreads();
    return s[0] + s[1] + s[2] + s[3];
}

struct BeamParams {
    const void* logits;
    const float* scores;      // [rows] or null
    const uint8_t* finished;  // [rows] or null
    const uint32_t* mask;     // or null
    uint64_t row_stride, mask_stride;
    uint32_t rows, groups, beams, vocab, k, pieces, end_token, normalize;
    // per (row, piece)
    uint64_t* list;   // [rows][pieces][k]: order of the logit << 32 | ~token, best first, 0 behind the last
    double* sum;      // [rows][pieces] sum of exp(x - peak)
    float* peak;      // [rows][pieces] largest admitted logit; -inf: none; NaN: a NaN among them
    uint32_t* out_parents;
    uint32_t* out_tokens;
    float* out_scores;
    uint32_t* out_counts;
};

// One piece (PIECE_THREADS * EACH logits) of one row, held in registers.  GROUPS maxima per thread narrow the piece to
// the logits that can be among its k largest: the k-th largest of all these maxima is reached by k logits.
template <typename V, int EACH, int GROUPS>
__global__ __launch_bounds__(PIECE_THREADS) void beam_piece_kernel(BeamParams p) {
    constexpr int WIDE = 16 / V::size, LOADS = EACH / WIDE, PIECE = PIECE_THREADS * EACH, CAP = 1024;
    __shared__ uint32_t s_max[PIECE_THREADS * GROUPS];
    __shared__ uint64_t s_list[CAP];
    __shared__ double s_sum[4];
    __shared__ uint32_t s_top[4], s_nan, s_n, s_cnt[8];
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const uint32_t row = blockIdx.x / p.pieces, piece = blockIdx.x % p.pieces;
    const size_t at = (size_t)row * p.pieces + piece;
    uint64_t* list = p.list + at * p.k;
    const bool ended = p.finished && p.finished[row];
    const float start = p.scores ? p.scores[row] : 0.0f;
    if (ended || !(start > -__builtin_inff())) {  // nothing of this row is looked at
        for (uint32_t i = t; i < p.k; i += PIECE_THREADS)
            list[i] = ended && piece == 0 && i == 0 ? ((uint64_t)f2ord(0.0f) << 32) | (uint32_t)~p.end_token : 0;
        if (t == 0) { p.sum[at] = 0.0; p.peak[at] = -__builtin_inff(); }
        return;
    }
    if (t == 0) { s_nan = 0; s_n = 0; }
    const typename V::bits* x = (const typename V::bits*)p.logits + (uint64_t)row * p.row_stride;
    const uint32_t* mask = p.mask ? p.mask + (uint64_t)row * p.mask_stride : nullptr;
    const uint32_t first = piece * PIECE;
    // order of every logit (0: not admitted, -inf or NaN)
    uint32_t key[EACH];
    bool nan = false;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const uint32_t tok = first + (j * PIECE_THREADS + t) * WIDE;
        u32x4 raw = {0, 0, 0, 0};
        typename V::bits one[WIDE];
        if (tok + WIDE <= p.vocab) {
            raw = *(const u32x4_any*)(x + tok);
            __builtin_memcpy(one, &raw, 16);
        } else {
#pragma unroll
            for (int w = 0; w < WIDE; ++w) one[w] = tok + w < p.vocab ? x[tok + w] : (typename V::bits)0;
        }
        const uint32_t bits = mask ? (tok < p.vocab ? mask[tok >> 5] >> (tok & 31) : 0) : ~0u;  // WIDE divides 32
#pragma unroll
        for (int w = 0; w < WIDE; ++w) {
            const bool in = tok + w < p.vocab && ((bits >> w) & 1);
            const float f = V::widen(one[w]);
            nan |= in && f != f;
            key[j * WIDE + w] = in && f > -__builtin_inff() ? f2ord(f + 0.0f) : 0;
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        uint32_t m = 0;
#pragma unroll
        for (int e = g * (EACH / GROUPS); e < (g + 1) * (EACH / GROUPS); ++e) m = max(m, key[e]);
        s_max[g * PIECE_THREADS + t] = m;
        top = max(top, m);
    }
    top = wave_max(top);
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    if (nan) s_nan = 1;
    top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
    const float peak = top ? ord2f(top) : -__builtin_inff();
    double sum = 0.0;
    if (p.normalize && top) {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            if (key[e]) sum += exp_below0((double)ord2f(key[e]) - (double)peak);
        sum = wave_sum(sum);
        if (lane == 0) s_sum[wave] = sum;
    }
    // the logits at or above the pivot
    const uint32_t pivot = max(kth_largest<4 * GROUPS>(s_max, p.k, lane), 1u);
#pragma unroll
    for (int e = 0; e < EACH; ++e)
        if (key[e] >= pivot) {
            const uint32_t i = atomicAdd(&s_n, 1u);
            const uint32_t tok = first + ((e / WIDE) * PIECE_THREADS + t) * WIDE + e % WIDE;
            if (i < CAP) s_list[i] = ((uint64_t)key[e] << 32) | (uint32_t)~tok;
        }
    __syncthreads();
    uint32_t n = s_n;
    if (t == 0) {
        p.sum[at] = p.normalize && top ? (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]) : 0.0;
        p.peak[at] = s_nan ? __uint_as_float(0x7fc00000u) : peak;
    }
    if (n > CAP) {
        // thousands of equal logits, or an order that puts all large ones into few threads: the k-th largest logit bit by
        // bit, then the lowest places among those that equal it
        uint32_t turn = 0, kth = 0, below = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t cand = kth | (1u << bit);
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < EACH; ++e) c += key[e] >= cand;
            if (block_count(c, s_cnt, turn++) >= p.k) kth = cand;
        }
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) c += key[e] > kth;
        const uint32_t need = p.k - block_count(c, s_cnt, turn++);  // >= 1 of those equal to it
        for (int bit = 13; bit >= 0; --bit) {  // the largest place that fewer than `need` of them lie below
            const uint32_t cand = below | (1u << bit);
            c = 0;
#pragma unroll
            for (int e = 0; e < EACH; ++e) c += key[e] == kth && ((e / WIDE) * PIECE_THREADS + t) * WIDE + e % WIDE < cand;
            if (block_count(c, s_cnt, turn++) < need) below = cand;
        }
        __syncthreads();
        if (t == 0) s_n = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const uint32_t place = ((e / WIDE) * PIECE_THREADS + t) * WIDE + e % WIDE;
            if (key[e] > kth || (key[e] == kth && place <= below))
                s_list[atomicAdd(&s_n, 1u)] = ((uint64_t)key[e] << 32) | (uint32_t)~(first + place);
        }
        __syncthreads();
        n = s_n;  // k
    }
    // their order by counting: the entries are all different
    for (uint32_t i = t; i < n; i += PIECE_THREADS) {
        const uint64_t mine = s_list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += s_list[j] > mine;
        if (rank < p.k) list[rank] = mine;
    }
    for (uint32_t i = n + t; i < p.k; i += PIECE_THREADS) list[i] = 0;
}

// One group: the logs of its rows' sums, the totals of what the pieces listed, and the k best of them.
template <int GROUPS>
__global__ __launch_bounds__(256) void beam_join_kernel(BeamParams p) {
    constexpr uint32_t CAP = 2048;
    __shared__ double s_lse[BEAMS_MAX];
    __shared__ float s_start[BEAMS_MAX];
    __shared__ uint32_t s_max[256 * GROUPS], s_n, s_cnt[8];
    __shared__ uint64_t s_ord[CAP], s_entry[CAP];
    __shared__ uint16_t s_beam[CAP];
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, group = blockIdx.x;
    const size_t row0 = (size_t)group * p.beams;
    for (uint32_t b = wave; b < p.beams; b += 4) {
        const size_t at = (row0 + b) * p.pieces;
        const bool ended = p.finished && p.finished[row0 + b];
        double lse = 0.0;
        if (p.normalize && !ended) {
            float m = -__builtin_inff();
            bool bad = false;
            for (uint32_t i = lane; i < p.pieces; i += 64) {
                const float v = p.peak[at + i];
                bad |= v != v;
                m = fmaxf(m, v);
            }
            for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            bad = __any(bad) || m == __builtin_inff();
            double s = 0.0;
            if (m > -__builtin_inff())
                for (uint32_t i = lane; i < p.pieces; i += 64) s += p.sum[at + i] * exp_below0((double)p.peak[at + i] - (double)m);
            s = wave_sum(s);
            lse = bad ? __longlong_as_double(0x7ff8000000000000ll) : (double)m + log(s);
        }
        if (lane == 0) {
            s_lse[b] = lse;
            s_start[b] = p.scores ? p.scores[row0 + b] : 0.0f;
        }
    }
    if (t == 0) s_n = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) s_max[g * 256 + t] = 0;
    __syncthreads();
    const uint64_t* list = p.list + row0 * p.pieces * p.k;
    const uint32_t per_row = p.pieces * p.k;
    const uint64_t slots = (uint64_t)p.beams * per_row;
    // order of the total, list entry and beam of a slot; an ended beam's entry holds a logit of 0 and no sum
    auto total_of = [&](uint64_t i, uint64_t* entry, uint32_t* beam) -> uint64_t {
        const uint64_t e = list[i];
        if (!e) return 0;
        const uint32_t b = slots >> 32 ? (uint32_t)(i / per_row) : (uint32_t)i / per_row;
        *entry = e;
        *beam = b;
        return order64((double)s_start[b] + ((double)ord2f((uint32_t)(e >> 32)) - s_lse[b]));
    };
    uint64_t entry = 0;
    uint32_t beam = 0;
    {
        uint32_t m[GROUPS] = {}, g = 0;
        for (uint64_t i = t; i < slots; i += 256) {
            const uint32_t h = (uint32_t)(total_of(i, &entry, &beam) >> 32);
#pragma unroll
            for (uint32_t q = 0; q < GROUPS; ++q)
                if (q == g) m[q] = max(m[q], h);
            g = g + 1 == GROUPS ? 0 : g + 1;
        }
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) s_max[q * 256 + t] = m[q];
    }
    __syncthreads();
    const uint32_t pivot = kth_largest<4 * GROUPS>(s_max, p.k, lane);
    auto keep = [&](uint64_t o) {
        const uint32_t at = atomicAdd(&s_n, 1u);
        if (at < CAP) { s_ord[at] = o; s_entry[at] = entry; s_beam[at] = (uint16_t)beam; }
    };
    for (uint64_t i = t; i < slots; i += 256) {
        const uint64_t o = total_of(i, &entry, &beam);
        if (o && (uint32_t)(o >> 32) >= pivot) keep(o);
    }
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
            for (uint64_t i = t; i < slots; i += 256) c += total_of(i, &entry, &beam) >= cand;
            if (block_count(c, s_cnt, turn++) >= p.k) kth = cand;
        }
        c = 0;
        for (uint64_t i = t; i < slots; i += 256) c += total_of(i, &entry, &beam) > kth;
        uint32_t need = p.k - block_count(c, s_cnt, turn++);
        for (int bit = 9; bit >= 0; --bit) {  // the largest beam that fewer than `need` of the equal ones lie before
            const uint32_t cand = last_beam | (1u << bit);
            c = 0;
            for (uint64_t i = t; i < slots; i += 256) c += total_of(i, &entry, &beam) == kth && beam < cand;
            if (block_count(c, s_cnt, turn++) < need) last_beam = cand;
        }
        c = 0;
        for (uint64_t i = t; i < slots; i += 256) c += total_of(i, &entry, &beam) == kth && beam < last_beam;
        need -= block_count(c, s_cnt, turn++);
        for (int bit = 63; bit >= 0; --bit) {  // entries count down: ~entry ascends
            const uint64_t cand = last | (1ull << bit);
            c = 0;
            for (uint64_t i = t; i < slots; i += 256) c += total_of(i, &entry, &beam) == kth && beam == last_beam && ~entry < cand;
            if (block_count(c, s_cnt, turn++) < need) last = cand;
        }
        __syncthreads();
        if (t == 0) s_n = 0;
        __syncthreads();
        for (uint64_t i = t; i < slots; i += 256) {
            const uint64_t o = total_of(i, &entry, &beam);
            if (o > kth || (o == kth && (beam < last_beam || (beam == last_beam && ~entry <= last)))) keep(o);
        }
        __syncthreads();
        n = s_n;  // k
    }
    uint32_t* parents = p.out_parents + (size_t)group * p.k;
    uint32_t* tokens = p.out_tokens + (size_t)group * p.k;
    float* scores = p.out_scores + (size_t)group * p.k;
    for (uint32_t i = t; i < n; i += 256) {
        const uint64_t o = s_ord[i], e = s_entry[i];
        const uint32_t b = s_beam[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j)
            rank += s_ord[j] > o || (s_ord[j] == o && (s_beam[j] < b || (s_beam[j] == b && s_entry[j] > e)));
        if (rank < p.k) {
            parents[rank] = b;
            tokens[rank] = (uint32_t)~(uint32_t)e;
            scores[rank] = (float)of_order64(o);
        }
    }
    for (uint32_t i = n + t; i < p.k; i += 256) {
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
template <typename V>
static void launch_pieces(const BeamParams& p, hipStream_t stream) {
    const dim3 grid(p.rows * p.pieces);
    if (p.k <= 64) hipLaunchKernelGGL((beam_piece_kernel<V, 32, 1>), grid, dim3(PIECE_THREADS), 0, stream, p);
    else hipLaunchKernelGGL((beam_piece_kernel<V, 32, 4>), grid, dim3(PIECE_THREADS), 0, stream, p);
}
constexpr uint32_t PIECE_LEN = PIECE_THREADS * 32;

static needle_hip_status states_check(const needle_beam_state* states, uint32_t n_states, uint64_t rows, uint64_t picks) {
    if (n_states && !states) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "states is null");
    if (n_states > STATES_MAX) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "at most %u states per call", STATES_MAX);
    struct Range { uint64_t first, second; } from[STATES_MAX] = {}, to[STATES_MAX] = {};  // first byte, last byte + 1
    for (uint32_t i = 0; i < n_states; ++i) {
        const needle_beam_state& s = states[i];
        if (s.outer == 0 || s.inner == 0 || s.bytes == 0) continue;
        if (!s.src || !s.dst) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "state %u has a null pointer", i);
        // rows, outer and inner runs of dst lie apart in one of their orders: no byte is written twice
        struct Axis { uint64_t n, stride; } ax[3] = {{s.outer, s.dst_outer_stride}, {picks, s.dst_row_stride}, {s.inner, s.dst_inner_stride}};
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
        from[i] = {(uint64_t)s.src, (uint64_t)s.src + reach};
        to[i] = {(uint64_t)s.dst, (uint64_t)s.dst + span};
    }
    for (uint32_t i = 0; i < n_states; ++i)
        for (uint32_t j = 0; j < n_states; ++j) {
            if (to[i].first < from[j].second && from[j].first < to[i].second)
                return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "dst of state %u overlaps src of state %u", i, j);
            if (i != j && to[i].first < to[j].second && to[j].first < to[i].second)
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

static needle_hip_status select_check(needle_hip_ctx* c, const needle_beam_params* q, const void* logits, const uint32_t* parents,
                                      const uint32_t* tokens, const float* scores, const uint32_t* counts) {
    if (!c || !q) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "null argument");
    if (!value_known(q->value)) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "unknown value type %d", q->value);
    if (q->reserved) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "reserved is not 0");
    ST_TRY(shape_check(q->groups, q->beams, q->k));
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
    const struct { const void* p; uint64_t n; } outs[4] = {{parents, np}, {tokens, np}, {scores, np}, {counts, (uint64_t)q->groups * 4}},
        ins[4] = {{logits, nl}, {q->scores, rows * 4}, {q->finished, rows}, {q->mask, nm}};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (ranges_meet(outs[i].p, outs[i].n, ins[j].p, ins[j].n) || (i != j && ranges_meet(outs[i].p, outs[i].n, outs[j].p, outs[j].n)))
                return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "an output overlaps another array");
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
    BeamParams p{};
    p.beams = q.beams; p.vocab = q.vocab; p.k = q.k; p.end_token = q.end_token; p.normalize = q.normalize != 0;
    p.row_stride = q.row_stride; p.mask_stride = q.mask_stride;
    p.pieces = (q.vocab + PIECE_LEN - 1) / PIECE_LEN;
    // a block of groups at a time: the pieces' lists stay within 256 MiB (one group's may be more), the grid within 2^22
    const uint64_t group_pieces = (uint64_t)q.beams * p.pieces, piece_bytes = (uint64_t)q.k * 8 + 12;
    uint64_t blk = std::min<uint64_t>((256ull << 20) / (group_pieces * piece_bytes), (1u << 22) / group_pieces);
    blk = std::max<uint64_t>(1, std::min<uint64_t>(blk, q.groups));
    HIP_TRY(c->scratch[7].ensure(blk * group_pieces * piece_bytes));
    p.list = c->scratch[7].as<uint64_t>();
    p.sum = (double*)(p.list + blk * group_pieces * q.k);
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
        case NEEDLE_VALUE_F32: launch_pieces<ValueF32>(p, c->stream); break;
        case NEEDLE_VALUE_F16: launch_pieces<ValueF16>(p, c->stream); break;
        default: launch_pieces<ValueBF16>(p, c->stream);
        }
        HIP_TRY(hipGetLastError());
        if (q.k <= 64) hipLaunchKernelGGL((beam_join_kernel<1>), dim3(p.groups), dim3(256), 0, c->stream, p);
        else hipLaunchKernelGGL((beam_join_kernel<4>), dim3(p.groups), dim3(256), 0, c->stream, p);
        HIP_TRY(hipGetLastError());
    }
    return NEEDLE_HIP_OK;
}

}  // namespace nh

using namespace nh;

extern "C" needle_hip_status needle_hip_beam_select_device(needle_hip_ctx* c, const needle_beam_params* q, const void* d_logits,
                                                           const needle_beam_state* states, uint32_t n_states, uint32_t* d_out_parents,
                                                           uint32_t* d_out_tokens, float* d_out_scores, uint32_t* d_out_counts) {
    ST_TRY(select_check(c, q, d_logits, d_out_parents, d_out_tokens, d_out_scores, d_out_counts));
    if (q->groups == 0) return NEEDLE_HIP_OK;
    const bool moves = n_states && q->k && q->beams;
    if (moves) ST_TRY(states_check(states, n_states, (uint64_t)q->groups * q->beams, (uint64_t)q->groups * q->k));
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    ST_TRY(select_enqueue(c, *q, d_logits, d_out_parents, d_out_tokens, d_out_scores, d_out_counts));
    if (moves) HIP_TRY(launch_moves(d_out_parents, q->groups, q->beams, q->k, states, n_states, c->n_cu, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}

extern "C" needle_hip_status needle_hip_beam_select(needle_hip_ctx* c, const needle_beam_params* q, const void* logits,
                                                    uint32_t* out_parents, uint32_t* out_tokens, float* out_scores, uint32_t* out_counts) {
    if (!c || !q) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "null argument");
    needle_beam_params h = *q;
    h.row_stride = h.vocab;
    const uint64_t words = ((uint64_t)h.vocab + 31) / 32;
    ST_TRY(select_check(c, &h, logits, out_parents, out_tokens, out_scores, out_counts));
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
    ST_TRY(states_check(states, n_states, (uint64_t)groups * beams, (uint64_t)groups * k));
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    HIP_TRY(launch_moves(d_parents, groups, beams, k, states, n_states, c->n_cu, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}
