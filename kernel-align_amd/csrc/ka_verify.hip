// Verification of drafted tokens: a drafter proposes up to K tokens per request, the target model scores the K + 1 positions
// in one forward pass, and the tokens are accepted or redrawn so that what comes out is distributed as the sampling operator
// would draw it from the target rows alone (speculative sampling).
//
//   P = W^p / Z^p, Q = W^q / Z^q      the rows' distributions after temperature, top-k and top-p, as integer masses: those of
//                                     the sampling kernels (Q is one-hot at the draft when there are no draft logits)
//   position j accepts d_j  iff  u_j Q(d_j) < P(d_j);  n = the first position that does not, or the number of drafts
//   ids[n] = inverse CDF, in index order, of max(P - Q, 0) (rejected) or of P (every draft accepted)
//
// Everything is decided as if on integers: u_j W^q Z^p < W^p Z^q (126 bits), residual masses max(W^p Z^q - W^q Z^p, 0) (102 bits
// each, 124 bits in sum).  A rejected draft with Q(d) > 0 always leaves a residual: P(d) <= u Q(d) < Q(d), both sum to one
// exactly, so some other entry has P > Q.  A draft that Q cannot have drawn (filtered out, or no entry at all) may meet P = Q:
// then the token is drawn from P.  Nothing depends on the order of a sum, on the batch or on the launch.
//
// The acceptance is evaluated in those integers.  The draw is first evaluated in fp64, with a bound of its error: each P_i =
// W^p_i / Z^p is off by 3 * 2^-53 of itself, R_i by 2^-51 (P_i + Q_i), and a sum of them, added in runs and trees of fewer than
// 2^12 terms, by 2^-41 in all (P and Q sum to one).  An entry whose prefix sums lie more than DRAW_MARGIN = 2^-38 on either side of u R is the
// integers' answer too; otherwise (about one draw in 10^6, and u = 0) the workgroup repeats the draw in 128-bit integers, two passes over the
// row by one workgroup: 64 requests x 4 drafts with u = 0 everywhere take 215 us instead of 80 with top-k and 480 instead of 91 without.
//
// Three launches, five where rows are split, no host synchronisation:
//   verify_split_top, verify_split_mass   few fp16 / fp32 rows without top-k only: maxima and masses by several workgroups per row
//   verify_rows    one workgroup per row that counts (target rows 0 .. len, draft rows 0 .. len - 1): the cut of the row's
//                  distribution, its total mass, the draft token's mass, the log-sum-exp of the raw row.  This is the pass over
//                  the data, 2 V (2 K + 1) bytes per request.
//   verify_shares  residual mass of every share of 256 vectors of the stopping position, a wavefront each
//   verify_draw    one workgroup per request: the share, the vector and the entry that hold the draw; all outputs
// Where top-p cuts inside a group of equal logits, the first r of the group survive, in index order.  verify_shares cannot know
// which those are: it counts the group's entries in its share and leaves the share's sum for either case, with the group or
// without it, and verify_draw, which sees all counts, picks one and evaluates the share again in which the r-th lies.
// The rows of the stopping position are read again by the last ones, from L2 / MALL as a rule.
#define KA_SAMPLING_THREADS 512
#include <stddef.h>

#include <atomic>
#include <type_traits>

#include "ka_sampling_common.h"
#include "ka_sampling_radix.h"

namespace ka {
namespace {

typedef unsigned __int128 u128;

constexpr int VERIFY_MAX_DRAFT = KA_VERIFY_MAX_DRAFT;
static_assert(VERIFY_MAX_DRAFT <= kWave, "one lane decides one position");
constexpr int64_t VERIFY_MAX_VOCAB = int64_t(1) << 22;           // below it: masses of 2^40 add up to less than 2^62
constexpr int64_t VERIFY_MAX_BATCH = 65535;                      // the second dimension of a grid
constexpr int64_t VERIFY_MAX_ROWS = (int64_t(1) << 32) / S_THREADS;  // below it: a grid of a workgroup per row
constexpr int SHARE_VECS = 256;    // 16-byte vectors of a row in one share; verify_draw has a thread for each
constexpr int SHARE_THREADS = 256;

// What verify_rows leaves about a row.
struct RowSummary {
    uint64_t z;         // integer mass of the survivors
    uint64_t w_draft;   // of which the drafted token has this (0: filtered out, or an id outside the vocabulary)
    double raw_sum;     // log-sum-exp of the raw row = raw_top + ln(raw_sum) (target rows, when asked for)
    float raw_top;
    uint32_t kmax, kcut, r_cut;  // see RowCut
    uint32_t raw_cut;   // key (unscaled) below which no entry survives; 0: not known, or no filter
    uint32_t pad;
};
static_assert(sizeof(RowSummary) == 48, "the workspace query counts 48 bytes per row");

// Residual mass of a share of the stopping position, by what becomes of the two rows' tie groups at their cuts.
struct ShareSums {
    double all;       // both groups survive
    double without_p; // the target's group does not
    double without_q; // the draft's group does not
    double neither;
    uint32_t ties_p, ties_q;  // entries of the groups; 0 where a group survives whole
};
static_assert(sizeof(ShareSums) == 40, "the workspace query counts 40 bytes per share");

// Of one part of a row that several workgroups work on (see verify_split_top).
struct SplitPart {
    uint64_t mass, raw;  // masses; exp(x - maximum) of the unscaled row in 2^-40
    uint32_t top, bad;   // largest key; an entry of 2^8 or more, or NaN
};
static_assert(sizeof(SplitPart) == 24, "the workspace query counts 24 bytes per part");

struct VerifyParams {
    const void *target, *draft;                          // draft may be null
    int64_t t_batch, t_pos, d_batch, d_pos;              // strides in elements
    const int64_t *draft_ids, *draft_lens;               // [B, K]; lens may be null (all K)
    const float *uniforms;                               // [B, K + 1]: acceptance, then the draw
    int32_t batch, k, vocab;
    float temperature, top_p;
    int32_t top_k;
    const float *temperature_rows, *top_p_rows;          // [B] each, or null
    const int32_t *top_k_rows;
    int64_t *out_ids, *out_accepted;
    float *out_policy;                                   // may be null
    RowSummary *rows;                                    // [B (K + 1)] target rows, then [B K] draft rows
    ShareSums *shares;                                   // [B, n_shares]
    int32_t n_shares, shares_per_group, vec_target, vec_draft;
    int32_t n_rows, split_parts, split_entries;          // rows; parts of a row that was worked on ahead (0: none), entries in each
    SplitPart *split;                                    // [rows, split_parts]
    uint64_t *split_bins;                                // [rows, HIST_BINS]
};

struct Filter { float temp; bool has_t; bool use_k; int top_k; bool use_p; float top_p; };
__device__ __forceinline__ Filter filter_of(const VerifyParams &p, int b) {
    Filter f{p.temperature, false, false, p.top_k, false, p.top_p};
    if (p.temperature_rows != nullptr) { f.temp = p.temperature_rows[b]; if (!(f.temp > 0.0f)) f.temp = 1.0f; }
    if (p.top_k_rows != nullptr) { f.top_k = p.top_k_rows[b]; if (f.top_k < 0) f.top_k = 0; }
    if (p.top_p_rows != nullptr) { f.top_p = p.top_p_rows[b]; if (!(f.top_p > 0.0f && f.top_p <= 1.0f)) f.top_p = 1.0f; }
    f.has_t = f.temp != 1.0f;
    f.use_k = f.top_k > 0 && f.top_k < p.vocab;
    f.use_p = f.top_p < 1.0f;
    return f;
}

__device__ __forceinline__ int draft_len(const VerifyParams &p, int b) {
    if (p.draft_lens == nullptr) return p.k;
    const int64_t n = p.draft_lens[b];
    return n < 0 ? 0 : (n > p.k ? p.k : int(n));
}
template <typename T> __device__ __forceinline__ const typename T::raw_t *target_row(const VerifyParams &p, int b, int j) {
    return static_cast<const typename T::raw_t *>(p.target) + int64_t(b) * p.t_batch + int64_t(j) * p.t_pos;
}
template <typename T> __device__ __forceinline__ const typename T::raw_t *draft_row(const VerifyParams &p, int b, int j) {
    return static_cast<const typename T::raw_t *>(p.draft) + int64_t(b) * p.d_batch + int64_t(j) * p.d_pos;
}

// A uniform as the sampling kernels take it: below 0 or NaN counts as 0, 1 and above as the largest number below 1.
__device__ __forceinline__ float clean_uniform(float u) {
    if (!(u >= 0.0f)) return 0.0f;
    return u >= 1.0f ? __uint_as_float(0x3f7fffffu) : u;
}
// u = mant * 2^-shift, 24 <= shift <= 149
__device__ __forceinline__ void split_uniform(float u, uint32_t &mant, int &shift) {
    const uint32_t b = __float_as_uint(u), e = (b >> 23) & 0xffu, m = b & 0x7fffffu;
    mant = e == 0 ? m : (m | 0x800000u);
    shift = e == 0 ? 149 : 150 - int(e);
}
// u * wq / zq < wp / zp, exactly.  w <= 2^40, z < 2^62: the products stay below 2^102, times the mantissa below 2^126.
__device__ __forceinline__ bool accepts(float u, uint64_t wp, uint64_t zp, uint64_t wq, uint64_t zq) {
    const u128 have = u128(wp) * zq;
    if (have == 0) return false;
    uint32_t mant;
    int shift;
    split_uniform(u, mant, shift);
    if (shift >= 128 || (have >> (128 - shift)) != 0) return true;  // have * 2^shift has at least 129 bits
    return u128(mant) * (u128(wq) * zp) < (have << shift);
}
// floor(u * r) for r < 2^124
__device__ __forceinline__ u128 floor_scale_wide(float u, u128 r) {
    uint32_t mant;
    int shift;
    split_uniform(u, mant, shift);
    // r = hi * 2^64 + lo: mant * r as three 64-bit limbs
    const u128 a = u128(mant) * uint64_t(r), b = u128(mant) * uint64_t(r >> 64) + uint64_t(a >> 64);
    // (b, low limb of a): b < 2^85
    if (shift >= 64) return shift - 64 >= 128 ? u128(0) : b >> (shift - 64);
    return (b << (64 - shift)) | (uint64_t(a) >> shift);
}

// The first position of request b that rejects its draft, or the number of drafts.  Called by whole wavefronts; every lane
// gets the result.
__device__ __forceinline__ int accepted_prefix(const VerifyParams &p, int b, int len) {
    const int j = int(threadIdx.x) & (kWave - 1);
    bool ok = false;
    if (j < len) {
        const RowSummary &t = p.rows[int64_t(b) * (p.k + 1) + j];
        uint64_t wq = 1, zq = 1;
        if (p.draft != nullptr) {
            const RowSummary &d = p.rows[int64_t(p.batch) * (p.k + 1) + int64_t(b) * p.k + j];
            wq = d.w_draft;
            zq = d.z;
        }
        ok = accepts(clean_uniform(p.uniforms[int64_t(b) * (p.k + 1) + j]), t.w_draft, t.z, wq, zq);
    }
    const uint64_t fails = ~__ballot(ok);
    const int first = fails == 0 ? kWave : __ffsll((long long)fails) - 1;
    return first < len ? first : len;
}

// One vector of entries from `base` on; zeros behind the row.
template <typename T>
__device__ __forceinline__ uint4 load_entries(const typename T::raw_t *row, bool vec, int vocab, int64_t base) {
    constexpr int EPV = T::kPerVec;
    if (vec && base + EPV <= vocab) return *reinterpret_cast<const uint4 *>(row + base);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < EPV; ++j)
        if (base + j < vocab) w[j * T::kBytes / 4] |= uint32_t(row[base + j]) << (T::kBytes == 2 ? 16 * (j & 1) : 0);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Entry j of a vector, j not known at compile time.
template <typename T> __device__ __forceinline__ typename T::raw_t entry_of(const uint4 &v, int j) {
    constexpr int HALF = T::kPerVec / 2;
    const uint64_t lo = (uint64_t(v.y) << 32) | v.x, hi = (uint64_t(v.w) << 32) | v.z;
    return typename T::raw_t((j & HALF ? hi : lo) >> (8 * T::kBytes * (j & (HALF - 1))));
}
// Bit j: entry base + j lies in the row and is not below `low` (NaN is not).
template <typename T> __device__ __forceinline__ uint32_t at_least(const uint4 &v, float low, int64_t base, int vocab) {
    float x[T::kPerVec];
    T::unpack(v, x);
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < T::kPerVec; ++j) bits |= !(x[j] < low) ? 1u << j : 0u;
    const int64_t room = vocab - base;
    return room >= T::kPerVec ? bits : (room <= 0 ? 0u : bits & ((1u << int(room)) - 1u));
}
// Bit j: entry base + j lies in the row and its scaled key is `key` (no entry below `low` has it).
template <typename T> __device__ __forceinline__ uint32_t ties_of(const uint4 &v, float low, int64_t base, int vocab, uint32_t key, const Filter &f) {
    uint32_t ties = 0;
#pragma unroll 1
    for (uint32_t left = at_least<T>(v, low, base, vocab); left != 0; left &= left - 1) {
        const int j = __ffs(left) - 1;
        if (elem_key<T>(entry_of<T>(v, j), f.temp, f.has_t) == key) ties |= 1u << j;
    }
    return ties;
}
// The value below which an unscaled entry does not survive (NaN compares as surviving: its key decides).
template <typename T> __device__ __forceinline__ float cut_value(uint32_t raw_cut) {
    return raw_cut == 0 ? -__builtin_inff() : value_of<T>(raw_cut);
}

// ---------------------------------------------------------------------------
// verify_rows
//
// A bf16 row has few distinct values, and everything a summary holds is a function of how often each occurs: one streaming
// pass counts the values of 2^-11 <= |x| < 2^8 in 4864 bins (19 KB of LDS, so that three workgroups share a CU and one row's
// tail runs under the reads of the others), lists the few smaller ones, and drops x <= -2^8, which has no mass next to an
// ordinary maximum.  Masses are then evaluated once per occupied bin instead of once per entry (by all threads where a sum
// over the whole row is needed), and one wavefront walks the bins from the largest value down to the cuts, 64 at a time.  Rows
// it cannot describe (values of 2^8 and above, NaN, a maximum or a cut among the small values, dropped values that would
// count) take the radix path.  Measured, bf16, 128,256 entries: 576 rows (64 requests x 4 drafts, 148 MB) 50 us, 2.9 TB/s, of which
// the stream takes about 30 (an atomic on LDS per entry) and the masses and the walk behind it, which all rows reach together, the rest;
// 2304 rows, of which about 56 % count: 106 us.  (A plain read of the 148 MB takes 21 us, and the sampling operator's short top-k route summarises
// 512 such rows in 28: most entries that are counted here do not survive.)  At the six wavefronts per SIMD that let three bf16
// workgroups share a CU, 30 registers are spilled; the fp16 and fp32 builds have 56 KB of LDS, two workgroups a CU.
// ---------------------------------------------------------------------------
constexpr uint32_t MAG_LOW = 0x3A00u, MAG_HIGH = 0x4380u;  // bits of 2^-11 and 2^8
constexpr int HIST_SIDE = int(MAG_HIGH - MAG_LOW);         // values of one sign: 19 octaves of 128
constexpr int HIST_BINS = 2 * HIST_SIDE;                   // ascending: negative values first
constexpr int HIST_POS = HIST_BINS + 1;                    // positions in descending order: positive bins, the small values, negative bins
constexpr int TINY_CAP = 1024;
constexpr int WINDOW = 512;                                // positions whose mass is kept: the walks to the cuts rarely leave them
constexpr uint32_t NO_KEY = 0;                             // no value of a row has this key

struct HistRow {
    uint32_t bin[HIST_BINS];
    uint16_t tiny[TINY_CAP];
    uint32_t n_tiny, n_zero, give_up, dropped, first;
    uint64_t sums[S_WAVES][3];  // per wavefront: mass of all entries, of the small ones, and raw_fix of these
    double raw_sums[S_WAVES];   // sum of exp(x - max) over the unscaled row's bins
    uint64_t win_mass[WINDOW];  // mass and scaled key of the positions from the first occupied one on
    uint32_t win_key[WINDOW];
    RowCut cut;
    uint32_t raw_cut, ok;
    double raw_sum;
    float raw_top;
};
// fp16 and fp32 rows: see coarse_cut
constexpr int LIST_CAP = 2048;
struct CoarseRow {
    union {
        uint32_t count[HIST_BINS];
        uint64_t mass[HIST_BINS];
    };
    alignas(16) uint32_t key[LIST_CAP];
    uint32_t sorted[LIST_CAP];
    uint32_t n_list, give_up, max_key, ok;
    uint64_t sums[S_WAVES][2];  // per wavefront: mass of all entries, and raw_fix of them
    float edge_low, edge_high;  // the list takes entries of [edge_low, edge_high)
    uint64_t before;            // mass above edge_high
    RowCut cut;
    double raw_sum;
    float raw_top;
};
template <typename T> struct VerifyShared {
    union {
        Shared sh;
        std::conditional_t<T::kDtype == KA_DTYPE_BF16, HistRow, CoarseRow> row;
    };
    PolicyLse lse;
    uint32_t ties_before;
};

__device__ __forceinline__ uint32_t raw_of_bin(int bin) {
    return bin >= HIST_SIDE ? MAG_LOW + uint32_t(bin - HIST_SIDE) : 0x8000u | (MAG_LOW + uint32_t(HIST_SIDE - 1 - bin));
}
__device__ __forceinline__ int bin_of_pos(int q) { return q < HIST_SIDE ? HIST_BINS - 1 - q : HIST_BINS - q; }

__device__ __forceinline__ uint64_t wave_sum_u64_of(uint64_t v) {
    const uint64_t inc = wave_incl_scan_u64(v);
    return (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(inc >> 32)), kWave - 1))) << 32) |
           uint32_t(__builtin_amdgcn_readlane(int(uint32_t(inc)), kWave - 1));
}

// exp(x - xmax) in 2^-40, rounded: sums of it do not depend on their order, and are off by V 2^-41 + 2^-22 of themselves.
__device__ __forceinline__ uint64_t raw_fix(float x, float xmax) {
    const double e = double(fast_exp2((x - xmax) * kLseLog2e)) + 4096.0;  // (its last bit is 2^-40)
    return uint64_t(__double_as_longlong(e)) & 0x000fffffffffffffull;
}
// Counts the row into h.bin / h.tiny.  A barrier must follow.
__device__ __forceinline__ void hist_count(HistRow &h, const uint16_t *rp, int vocab) {
    const int tid = threadIdx.x;
    uint32_t zeros = 0, high = 0, low = 0;
    // m = magnitude bits - MAG_LOW (as an unsigned number: below the range wraps to the top), sign = 0 or all ones
    auto add = [&](uint32_t m, uint32_t sign) { if (m < uint32_t(HIST_SIDE)) atomicAdd(&h.bin[HIST_SIDE + int(m ^ sign)], 1u); };
    auto odd = [&](uint32_t x) {  // |x| outside the bins
        const uint32_t mag = x & 0x7fffu;
        if (mag - MAG_LOW < uint32_t(HIST_SIDE)) return;
        if (mag == 0) ++zeros;
        else if (mag < MAG_LOW) {
            const uint32_t at = atomicAdd(&h.n_tiny, 1u);
            if (at < uint32_t(TINY_CAP)) h.tiny[at] = uint16_t(x);
        } else if ((x & 0x8000u) == 0 || mag > 0x7f80u) high = 1;
        else low = 1;
    };
    auto one = [&](uint32_t x) {
        add((x & 0x7fffu) - MAG_LOW, (x & 0x8000u) ? ~0u : 0u);
        odd(x);
    };
    int head = int((16 - (reinterpret_cast<uintptr_t>(rp) & 15)) & 15) / 2;  // entries before the first whole vector
    head = head < vocab ? head : vocab;
    if (tid < head) one(rp[tid]);
    const uint4 *vp = reinterpret_cast<const uint4 *>(rp + head);
    const int nvec = (vocab - head) / 8;
    constexpr int U = 8;  // loads in flight per lane
    for (int v = tid; v < nvec; v += U * S_THREADS) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = v + u * S_THREADS < nvec ? load_stream(vp + v + u * S_THREADS) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (v + u * S_THREADS >= nvec) continue;
            const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
            uint32_t worst = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t m0 = (w[j] & 0x7fffu) - MAG_LOW, m1 = ((w[j] >> 16) & 0x7fffu) - MAG_LOW;
                worst = m0 > worst ? m0 : worst;
                worst = m1 > worst ? m1 : worst;
                add(m0, uint32_t(int32_t(w[j] << 16) >> 31));
                add(m1, uint32_t(int32_t(w[j]) >> 31));
            }
            if (worst >= uint32_t(HIST_SIDE)) {  // rare: small values, zeros, masked entries
                uint4 r = q[u];
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    odd(r.x & 0xffffu);
                    odd(r.x >> 16);
                    r.x = r.y;
                    r.y = r.z;
                    r.z = r.w;
                }
            }
        }
    }
    const int i = head + nvec * 8 + tid;
    if (i < vocab) one(rp[i]);
    if (zeros) atomicAdd(&h.n_zero, zeros);
    if (high) h.give_up = 1;
    if (low) h.dropped = 1;
}

// False: the row needs the radix path (nothing is decided).  h.cut, h.raw_cut and (with want_lse) h.raw_sum, h.raw_top hold the result.
__device__ __forceinline__ bool hist_cut(HistRow &h, const uint16_t *rp, int vocab, const Filter &f, bool want_lse) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    for (int i = tid; i < HIST_BINS; i += S_THREADS) h.bin[i] = 0;
    if (tid == 0) { h.n_tiny = h.n_zero = h.give_up = h.dropped = 0; h.first = HIST_POS; h.ok = 0; }
    __syncthreads();
    hist_count(h, rp, vocab);
    __syncthreads();
    const uint32_t n_tiny = h.n_tiny, n_zero = h.n_zero, n_mid = n_tiny + n_zero;
    if (h.give_up != 0 || n_tiny > uint32_t(TINY_CAP)) return false;
    auto key_of_raw = [&](uint32_t raw) { return elem_key<Bf16>(uint16_t(raw), f.temp, f.has_t); };
    auto count_at = [&](int q) -> uint32_t { return q >= HIST_POS ? 0u : (q == HIST_SIDE ? n_mid : h.bin[bin_of_pos(q)]); };
    {   // the largest value
        int mine = HIST_POS;
        for (int q = tid; q < HIST_POS && mine == HIST_POS; q += S_THREADS)
            if (count_at(q) != 0) mine = q;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            const int o = __shfl_xor(mine, off, kWave);
            mine = o < mine ? o : mine;
        }
        if (lane == 0) atomicMin(&h.first, uint32_t(mine));
    }
    __syncthreads();
    const int first = int(h.first);
    if (first == HIST_SIDE || first == HIST_POS) return false;
    const uint32_t raw_max = raw_of_bin(bin_of_pos(first));
    const uint32_t kmax = key_of_raw(raw_max);
    const float vmax = value_of<Bf16>(kmax), xmax = Bf16::widen(uint16_t(raw_max));
    auto weight_of = [&](uint32_t key) { return weight_fix(key == kmax ? 0.0f : value_of<Bf16>(key) - vmax); };
    // ---- masses: of all positions where a total is needed, else of the window -------------------
    const bool total = !f.use_k;
    {
        uint64_t all = 0, mid = 0, mid_raw = 0;
        double raw_sum = 0.0;
        // (without branches on empty bins, two at a time: the chain of fused multiply-adds is what takes the time)
        const int end = total ? HIST_POS : (first + WINDOW < HIST_POS ? first + WINDOW : HIST_POS);
#pragma unroll 2
        for (int q = first + tid; q < end; q += S_THREADS) {
            const uint32_t c = q == HIST_SIDE ? 0u : count_at(q);
            const uint32_t key = key_of_raw(raw_of_bin(bin_of_pos(q == HIST_SIDE ? first : q)));
            const uint64_t w = weight_of(key) * c;
            all += w;
            if (q < first + WINDOW) {
                h.win_mass[q - first] = w;
                h.win_key[q - first] = c != 0 ? key : NO_KEY;
            }
        }
        if (want_lse) {  // (fp32 exponentials, off by 2^-22 each: ample for a log-probability in fp32)
#pragma unroll 2
            for (int q = first + tid; q < HIST_POS; q += S_THREADS)
                if (q != HIST_SIDE) raw_sum += double(float(count_at(q)) * fast_exp2((Bf16::widen(uint16_t(raw_of_bin(bin_of_pos(q)))) - xmax) * kLseLog2e));
        }
        if (total || want_lse) {
#pragma unroll 1
            for (int i = tid; i <= int(n_tiny); i += S_THREADS) {  // the small values, then zero
                const uint32_t c = i < int(n_tiny) ? 1u : n_zero;
                const uint32_t raw = i < int(n_tiny) ? uint32_t(h.tiny[i]) : 0u;
                if (total) mid += weight_of(key_of_raw(raw)) * c;
                if (want_lse) mid_raw += raw_fix(Bf16::widen(uint16_t(raw)), xmax) * c;  // (integers: the list's order is the atomics')
            }
            all = wave_sum_u64_of(all);
            mid = wave_sum_u64_of(mid);
            mid_raw = wave_sum_u64_of(mid_raw);
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) raw_sum += __shfl_xor(raw_sum, off, kWave);
            if (lane == 0) {
                h.sums[wave][0] = all;
                h.sums[wave][1] = mid;
                h.sums[wave][2] = mid_raw;
                h.raw_sums[wave] = raw_sum;
            }
        }
        __syncthreads();
    }
    if (wave != 0) {
        __syncthreads();  // the first wavefront's result
        return h.ok != 0;
    }
    // ---- the first wavefront finishes the row --------------------------------------------------
    uint64_t z_all = 0, z_mid = 0, mid_raw = 0;
    double raw_sum = 0.0;
    if (total || want_lse)
        for (int w = 0; w < S_WAVES; ++w) {
            z_all += h.sums[w][0];
            z_mid += h.sums[w][1];
            mid_raw += h.sums[w][2];
            raw_sum += h.raw_sums[w];
        }
    z_all += z_mid;
    raw_sum += double(mid_raw) * 0x1p-40;
    const bool dropped = h.dropped != 0;
    uint32_t key_dropped = 0, key_tiny = 0, key_tiny_neg = 0;
    bool ok = true;
    if (dropped) {
        key_dropped = key_of_raw(0x8000u | MAG_HIGH);
        // (a temperature that takes every value of the row to -infinity makes them all its maximum)
        ok = weight_of(key_dropped) == 0 && weight_fix(-256.0f - xmax) == 0;
    }
    if (f.use_k || f.use_p) {
        key_tiny = key_of_raw(MAG_LOW - 1);
        key_tiny_neg = key_of_raw(0x8000u | (MAG_LOW - 1));
    }
    // a cut that shares its scaled value with entries that are not binned (a temperature that folds values together)
    auto shared_value = [&](uint32_t key, int q) {
        return (dropped && key <= key_dropped) || (n_mid > 0 && (q < HIST_SIDE ? key <= key_tiny : key >= key_tiny_neg));
    };
    RowCut cut{kmax, 0u, 0u, 0xffffffffu, z_all};
    uint32_t raw_cut = 0;
    auto last_u64 = [&](uint64_t v) {
        return (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), kWave - 1))) << 32) |
               uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), kWave - 1));
    };
    if (ok && f.use_k) {  // the position that holds the top_k-th largest entry
        uint32_t upto = 0;
        int kpos = -1;
        for (int q0 = first; q0 < HIST_POS && kpos < 0; q0 += kWave) {
            const uint32_t inc = upto + wave_incl_scan_u32(count_at(q0 + lane));
            const uint64_t reached = __ballot(inc >= uint32_t(f.top_k));
            if (reached != 0) kpos = q0 + __ffsll((long long)reached) - 1;
            upto = uint32_t(__builtin_amdgcn_readlane(int(inc), kWave - 1));
        }
        if (kpos < 0 || kpos == HIST_SIDE) ok = false;
        else {
            cut.kstar = cut.kcut = key_of_raw(raw_of_bin(bin_of_pos(kpos)));
            ok = !shared_value(cut.kstar, kpos);
            if (kpos > HIST_SIDE && n_mid > 0) ok = false;  // the small values would be among the survivors without a total
        }
    }
    // Key (NO_KEY: empty, the small values or below the top-k cut), count and mass of one position.
    auto position = [&](int q, uint32_t &key, uint32_t &c, uint64_t &m) {
        c = count_at(q);
        key = NO_KEY;
        m = 0;
        if (c == 0) return;
        if (q == HIST_SIDE) { m = z_mid; return; }
        key = q < first + WINDOW ? h.win_key[q - first] : key_of_raw(raw_of_bin(bin_of_pos(q)));
        if (key < cut.kstar) { key = NO_KEY; c = 0; return; }
        m = q < first + WINDOW ? h.win_mass[q - first] : weight_of(key) * c;
    };
    if (ok && f.use_k) {  // mass of the survivors of top-k: up to the first step with an entry below the cut
        uint64_t z = 0;
        for (int q0 = first; q0 < HIST_POS; q0 += kWave) {
            uint32_t key, c;
            uint64_t m;
            position(q0 + lane, key, c, m);
            z += wave_sum_u64_of(m);
            const bool below = q0 + lane < HIST_POS && count_at(q0 + lane) != 0 && key == NO_KEY;
            const uint64_t alive = __ballot(key != NO_KEY);
            if (alive != 0) raw_cut = raw_of_bin(bin_of_pos(q0 + 63 - __builtin_clzll(alive)));
            if (__ballot(below) != 0) break;
        }
        cut.z = z;
    }
    if (ok && f.use_p) {
        const uint64_t theta = floor_scale(f.top_p, cut.z);
        int best = -1;
        uint64_t run = 0;
        for (int q0 = first; q0 < HIST_POS && run <= theta; q0 += kWave) {
            uint32_t key, c;
            uint64_t m;
            position(q0 + lane, key, c, m);
            const uint64_t inc = wave_incl_scan_u64(m);
            const uint64_t in = __ballot(c != 0 && run + inc - m <= theta);
            if (in != 0) best = q0 + 63 - __builtin_clzll(in);
            run += last_u64(inc);
        }
        ok = best != HIST_SIDE;
        if (ok) {
            cut.kcut = key_of_raw(raw_of_bin(bin_of_pos(best)));
            ok = !shared_value(cut.kcut, best);
        }
        if (ok) {
            uint64_t before = 0;
            uint32_t n_cut = 0;
            run = 0;
            for (int q0 = first; q0 < HIST_POS; q0 += kWave) {
                uint32_t key, c;
                uint64_t m;
                position(q0 + lane, key, c, m);
                const uint64_t inc = wave_incl_scan_u64(m);
                const uint64_t group = __ballot(key == cut.kcut);
                if (group != 0) {
                    const uint64_t excl = run + inc - m;
                    if (n_cut == 0) {
                        const int l = __ffsll((long long)group) - 1;
                        before = (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(excl >> 32)), l))) << 32) |
                                 uint32_t(__builtin_amdgcn_readlane(int(uint32_t(excl)), l));
                    }
                    n_cut += uint32_t(__builtin_amdgcn_readlane(int(wave_incl_scan_u32(key == cut.kcut ? c : 0u)), kWave - 1));
                    raw_cut = raw_of_bin(bin_of_pos(q0 + 63 - __builtin_clzll(group)));
                }
                if (__ballot(q0 + lane > best && count_at(q0 + lane) != 0 && key != cut.kcut) != 0) break;  // behind the group
                run += last_u64(inc);
            }
            const uint64_t w_cut = weight_of(cut.kcut);
            uint64_t r = n_cut;
            if (w_cut > 0) {
                const uint64_t fit = (theta - before) / w_cut + 1;  // entries t with before + t * w <= theta
                r = fit < r ? fit : r;
            }
            cut.r_cut = r == n_cut ? 0xffffffffu : uint32_t(r);
            cut.z = before + r * w_cut;
        }
    }
    if (lane == 0) {
        h.cut = cut;
        h.raw_cut = f.use_k || f.use_p ? masked_key<Bf16>(Bf16::widen(uint16_t(raw_cut))) : 0u;
        h.raw_sum = raw_sum;
        h.raw_top = xmax;
        h.ok = ok ? 1u : 0u;
    }
    __syncthreads();
    return ok;
}

// The smallest unscaled key whose scaled value reaches kcut, by all lanes of the wavefront at once: near kcut's value times
// the temperature.  0 where it is not found there (underflow, infinities): the later passes then scale every entry.
template <typename T> __device__ __forceinline__ uint32_t raw_key_of_cut(uint32_t kcut, float temp, bool has_t) {
    if (!has_t || kcut == 0) return kcut;
    const uint32_t near = masked_key<T>(value_of<T>(kcut) * temp);
    const int lane = int(threadIdx.x) & (kWave - 1);
    const uint32_t mine = near + uint32_t(lane - kWave / 2) * key_step<T>();
    const float x = value_of<T>(mine);
    const uint64_t reach = __ballot(x == x && elem_key<T>(raw_of_key<T>(mine), temp, true) >= kcut);
    // a run of lanes up to the last one, not all of them
    if (reach == 0 || reach == ~uint64_t(0) || (reach >> 63) == 0) return 0;
    const int low = __ffsll((long long)reach) - 1;
    if ((reach >> low) != (~uint64_t(0) >> low)) return 0;
    return near + uint32_t(low - kWave / 2) * key_step<T>();
}

// ---------------------------------------------------------------------------
// fp16 and fp32 rows have too many values for a bin each.  The same bins, of the values cut to bf16, locate the cut; the
// entries of the bins around it (about top_k of them, or a few hundred) then go to a list, are sorted, and decide as in the
// definition.  No filter: the maximum, then the masses (two passes over the row).  Top-k: counts, then the list (two).  Top-p
// alone: the maximum, the mass of every bin, the list (three).  What does not fit (values of 2^8 and above, NaN, a cut among
// values below 2^-11 or at the edge of the list, more than 2048 entries in it) takes the radix path.
// ---------------------------------------------------------------------------
// f(entry) for every entry of the row by the whole block, in any order; eight vectors in flight per lane, any alignment.
template <typename T, typename F> __device__ __forceinline__ void each_entry(const typename T::raw_t *rp, int vocab, F &&f) {
    constexpr int EPV = T::kPerVec, U = 8;
    const int tid = threadIdx.x;
    int head = int((16 - (reinterpret_cast<uintptr_t>(rp) & 15)) & 15) / T::kBytes;
    head = head < vocab ? head : vocab;
    const int nvec = (vocab - head) / EPV, tail = head + nvec * EPV + tid;
    if (tid < head) f(rp[tid]);
    if (tail < vocab) f(rp[tail]);
    const uint4 *vp = reinterpret_cast<const uint4 *>(rp + head);
    for (int v = tid; v < nvec; v += U * S_THREADS) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = vp[v + u * S_THREADS < nvec ? v + u * S_THREADS : v];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (v + u * S_THREADS >= nvec) continue;
#pragma unroll
            for (int j = 0; j < EPV; ++j) f(entry_of<T>(q[u], j));
        }
    }
}

// Bin of a value, or HIST_BINS (small, zero), HIST_BINS + 1 (-2^8 and below), HIST_BINS + 2 (2^8 and above, NaN).
__device__ __forceinline__ int coarse_bin(float x) {
    const uint32_t b = __float_as_uint(x), mag = (b >> 16) & 0x7fffu, m = mag - MAG_LOW;
    if (m < uint32_t(HIST_SIDE)) return HIST_SIDE + int(m ^ uint32_t(int32_t(b) >> 31));
    if (mag < MAG_LOW) return HIST_BINS;
    return int32_t(b) < 0 && x == x ? HIST_BINS + 1 : HIST_BINS + 2;
}
// Largest value, in magnitude order of its sign, that a bin begins with (the bins are of values cut towards zero).
__device__ __forceinline__ float bin_value(int bin) { return __uint_as_float(raw_of_bin(bin) << 16); }
// Bins b .. hold the values from lower_edge(b) on.
__device__ __forceinline__ float lower_edge(int bin) {
    if (bin <= 0) return -256.0f;
    if (bin > HIST_BINS - 1) return 256.0f;
    // a negative bin holds (next bin down's value, its own value]: its lower edge is just above the value of the bin below
    return bin >= HIST_SIDE ? bin_value(bin) : __uint_as_float(__float_as_uint(bin_value(bin - 1)) - 1u);
}

// The maxima at which the bins describe a row.
__device__ __forceinline__ bool coarse_top(float xmax) { return (xmax >= 0x1p-11f || xmax <= -0x1p-11f) && xmax > -256.0f && xmax < 256.0f; }
// Mass and raw_fix of entries of a row, and the bins' masses (added to `bins` where `use_p`).
template <typename T>
__device__ __forceinline__ void coarse_masses(const typename T::raw_t *rp, int count, const Filter &f, bool want_lse, float xmax, uint32_t kmax,
                                              uint64_t *bins, uint64_t &all, uint64_t &raw) {
    const float vmax = value_of<T>(kmax);
    each_entry<T>(rp, count, [&](typename T::raw_t r) {
        const float x = T::widen(r);
        if (want_lse) raw += raw_fix(x, xmax);
        const uint32_t key = elem_key<T>(r, f.temp, f.has_t);
        const uint64_t w = weight_fix(key == kmax ? 0.0f : value_of<T>(key) - vmax);
        all += w;
        if (f.use_p && w != 0) {
            const int bin = coarse_bin(x);
            if (bin < HIST_BINS) atomicAdd(reinterpret_cast<unsigned long long *>(&bins[bin]), (unsigned long long)w);
        }
    });
}
// Maximum and flag over the parts of a row, in every lane of the wavefront.
__device__ __forceinline__ void split_top(const SplitPart *parts, int n, uint32_t &top, uint32_t &bad) {
    top = bad = 0;
    for (int i = int(threadIdx.x) & (kWave - 1); i < n; i += kWave) {
        top = parts[i].top > top ? parts[i].top : top;
        bad |= parts[i].bad;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const uint32_t o = __shfl_xor(top, off, kWave);
        top = o > top ? o : top;
        bad |= __shfl_xor(bad, off, kWave);
    }
}

// `parts`: what verify_split_top and verify_split_mass found about the row (n_parts of them, and its bins), or null.
template <typename T>
__device__ __forceinline__ bool coarse_cut(CoarseRow &h, const typename T::raw_t *rp, int vocab, const Filter &f, bool want_lse,
                                           const SplitPart *parts, int n_parts, const uint64_t *bins) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const bool ahead = parts != nullptr;  // (never with top-k)
    for (int i = tid; i < HIST_BINS; i += S_THREADS) h.mass[i] = ahead && f.use_p ? bins[i] : 0;
    if (tid == 0) { h.n_list = h.give_up = h.max_key = h.ok = 0; }
    __syncthreads();
    auto last_u64 = [&](uint64_t v) {
        return (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), kWave - 1))) << 32) |
               uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), kWave - 1));
    };
    // ---- first pass: the maximum, and with top-k the counts ----------------------------------
    if (ahead) {
        uint32_t top, bad;
        split_top(parts, n_parts, top, bad);
        if (tid == 0) { h.max_key = top; h.give_up = bad; }
    } else {
        uint32_t top = 0, bad = 0;
        each_entry<T>(rp, vocab, [&](typename T::raw_t raw) {
            const float x = T::widen(raw);
            const uint32_t key = masked_key<T>(x);
            top = key > top && x == x ? key : top;
            bad |= !(x < 256.0f) ? 1u : 0u;
            if (f.use_k) {
                const int bin = coarse_bin(x);
                if (bin < HIST_BINS) atomicAdd(&h.count[bin], 1u);
            }
        });
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            const uint32_t o = __shfl_xor(top, off, kWave);
            top = o > top ? o : top;
        }
        if (lane == 0) atomicMax(&h.max_key, top);
        if (bad) h.give_up = 1;
    }
    __syncthreads();
    const float xmax = value_of<T>(h.max_key);
    if (h.give_up != 0 || h.max_key == 0 || !coarse_top(xmax)) return false;
    const uint32_t kmax = elem_key<T>(raw_of_key<T>(h.max_key), f.temp, f.has_t);
    const float vmax = value_of<T>(kmax);
    auto weight_of = [&](uint32_t key) { return weight_fix(key == kmax ? 0.0f : value_of<T>(key) - vmax); };
    const int top_bin = coarse_bin(xmax);
    if (f.use_k) {
        // ---- the bin of the top_k-th largest entry; the list reaches one bin further ----------
        if (wave == 0) {
            uint32_t upto = 0;
            int found = -1;
            for (int b0 = top_bin; b0 >= 0 && found < 0; b0 -= kWave) {
                const int b = b0 - lane;
                const uint32_t inc = upto + wave_incl_scan_u32(b >= 0 ? h.count[b] : 0u);
                const uint64_t reached = __ballot(inc >= uint32_t(f.top_k));
                if (reached != 0) found = b0 - (__ffsll((long long)reached) - 1);
                upto = uint32_t(__builtin_amdgcn_readlane(int(inc), kWave - 1));
                // (past the smallest positive values lie entries that are not counted)
                if (found < HIST_SIDE && top_bin >= HIST_SIDE && b0 - kWave < HIST_SIDE) break;
            }
            if (lane == 0) {
                const bool side = found >= 0 && (found > HIST_SIDE || (found < HIST_SIDE && top_bin < HIST_SIDE && found > 0));
                h.ok = side ? 1u : 0u;
                h.edge_low = side ? lower_edge(found - 1) : 0.0f;
                h.edge_high = 256.0f;
                h.before = 0;
            }
        }
        __syncthreads();
        if (h.ok == 0) return false;
    }
    // ---- second pass: the list (top-k), or the masses -----------------------------------------
    uint64_t z_all = 0;
    double raw_sum = 0.0;
    {
        uint64_t all = 0, raw = 0;
        const float low = f.use_k ? h.edge_low : 0.0f;
        if (ahead) {
            for (int i = tid; i < n_parts; i += S_THREADS) {
                all += parts[i].mass;
                raw += parts[i].raw;
            }
        } else if (f.use_k) {
            each_entry<T>(rp, vocab, [&](typename T::raw_t r) {
                const float x = T::widen(r);
                if (want_lse) raw += raw_fix(x, xmax);
                if (x >= low) {
                    const uint32_t at = atomicAdd(&h.n_list, 1u);
                    if (at < uint32_t(LIST_CAP)) h.key[at] = elem_key<T>(r, f.temp, f.has_t);
                }
            });
        } else {
            coarse_masses<T>(rp, vocab, f, want_lse, xmax, kmax, h.mass, all, raw);
        }
        all = wave_sum_u64_of(all);
        raw = wave_sum_u64_of(raw);
        if (lane == 0) {
            h.sums[wave][0] = all;
            h.sums[wave][1] = raw;
        }
        __syncthreads();
        raw = 0;
        for (int w = 0; w < S_WAVES; ++w) {
            z_all += h.sums[w][0];
            raw += h.sums[w][1];
        }
        raw_sum = double(raw) * 0x1p-40;
        if (f.use_p && !f.use_k) {
            // ---- the bin where the mass before an entry passes theta; the list: it and its two neighbours ----
            if (wave == 0) {
                const uint64_t theta = floor_scale(f.top_p, z_all);
                uint64_t run = 0, before = 0;
                int found = -1;
                for (int b0 = top_bin; b0 >= 0 && found < 0; b0 -= kWave) {
                    const int b = b0 - lane;
                    const uint64_t m = b >= 0 ? h.mass[b] : 0ull;
                    const uint64_t inc = run + wave_incl_scan_u64(m);
                    const uint64_t passed = __ballot(inc > theta);  // the last entry kept lies in the first of these
                    if (passed != 0) {
                        const int l = __ffsll((long long)passed) - 1;
                        found = b0 - l;
                        const uint64_t at = inc - m;
                        before = (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(at >> 32)), l))) << 32) |
                                 uint32_t(__builtin_amdgcn_readlane(int(uint32_t(at)), l));
                    }
                    run = last_u64(inc);
                    if (found < HIST_SIDE && top_bin >= HIST_SIDE && b0 - kWave < HIST_SIDE) break;
                }
                if (lane == 0) {
                    const bool side = found >= 0 && (found > HIST_SIDE || (found < HIST_SIDE && top_bin < HIST_SIDE && found > 0));
                    // (one bin up, unless that is another sign's)
                    const bool up = side && found + 1 < HIST_BINS && found + 1 != HIST_SIDE;
                    h.ok = side ? 1u : 0u;
                    h.edge_low = side ? lower_edge(found - 1) : 0.0f;
                    h.edge_high = side ? lower_edge(up ? found + 2 : found + 1) : 0.0f;
                    if (side && found + 1 == HIST_SIDE) h.edge_high = 0.0f;
                    h.before = before - (up ? h.mass[found + 1] : 0ull);
                }
            }
            __syncthreads();
            if (h.ok == 0) return false;
            const float lo = h.edge_low, hi = h.edge_high;
            each_entry<T>(rp, vocab, [&](typename T::raw_t raw) {
                const float x = T::widen(raw);
                if (x >= lo && x < hi) {
                    const uint32_t at = atomicAdd(&h.n_list, 1u);
                    if (at < uint32_t(LIST_CAP)) h.key[at] = elem_key<T>(raw, f.temp, f.has_t);
                }
            });
            __syncthreads();
        }
    }
    RowCut cut{kmax, 0u, 0u, 0xffffffffu, z_all};
    bool ok = true;
    if (f.use_k || f.use_p) {
        const uint32_t n = h.n_list;
        if (n > uint32_t(LIST_CAP) || n == 0 || (f.use_k && n < uint32_t(f.top_k))) return false;
        // ---- sorted by key, descending (equal keys in any order: they have equal masses) ---------
        if (tid < 4 && n + uint32_t(tid) < uint32_t(LIST_CAP)) h.key[n + uint32_t(tid)] = NO_KEY;  // up to a multiple of four
        __syncthreads();
        for (uint32_t i = uint32_t(tid); i < n; i += S_THREADS) {
            const uint32_t k = h.key[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < n; j += 4) {
                const uint4 o = *reinterpret_cast<const uint4 *>(h.key + j);
                rank += (o.x > k || (o.x == k && j < i) ? 1u : 0u) + (o.y > k || (o.y == k && j + 1 < i) ? 1u : 0u) +
                        (o.z > k || (o.z == k && j + 2 < i) ? 1u : 0u) + (o.w > k || (o.w == k && j + 3 < i) ? 1u : 0u);
            }
            h.sorted[rank] = k;
        }
        __syncthreads();
        if (wave != 0) {
            __syncthreads();  // the first wavefront's result
            return h.ok != 0;
        }
        // a group at the list's lower end may go on behind it
        const uint32_t key_edge = masked_key<T>(h.edge_low) <= key_step<T>() ? 0u : elem_key<T>(raw_of_key<T>(masked_key<T>(h.edge_low)), f.temp, f.has_t);
        const uint32_t key_high = h.edge_high < 256.0f ? elem_key<T>(raw_of_key<T>(masked_key<T>(h.edge_high)), f.temp, f.has_t) : 0xffffffffu;
        uint64_t z = z_all;
        uint32_t na = n;  // entries of the list that survive top-k
        if (f.use_k) {
            cut.kstar = cut.kcut = h.sorted[f.top_k - 1];
            ok = cut.kstar > key_edge;
            z = 0;
            na = 0;
            for (uint32_t i0 = 0; i0 < n; i0 += kWave) {
                const uint32_t i = i0 + uint32_t(lane);
                const bool in = i < n && h.sorted[i] >= cut.kstar;
                z += wave_sum_u64_of(in ? weight_of(h.sorted[i]) : 0ull);
                const uint32_t here = uint32_t(__popcll(__ballot(in)));
                na += here;
                if (here < uint32_t(kWave)) break;
            }
            cut.z = z;
        }
        if (f.use_p && ok) {
            const uint64_t theta = floor_scale(f.top_p, z);
            uint64_t run = h.before;
            int best = -1;
            for (uint32_t i0 = 0; i0 < na && run <= theta; i0 += kWave) {
                const uint32_t i = i0 + uint32_t(lane);
                const uint64_t m = i < na ? weight_of(h.sorted[i]) : 0ull;
                const uint64_t inc = run + wave_incl_scan_u64(m);
                const uint64_t in = __ballot(i < na && inc - m <= theta);
                if (in != 0) best = int(i0) + 63 - __builtin_clzll(in);
                run = last_u64(inc);
            }
            ok = best >= 0;
            if (ok) {
                cut.kcut = h.sorted[best];
                ok = cut.kcut > key_edge && cut.kcut < key_high;
            }
            if (ok) {
                uint64_t before = h.before;
                uint32_t n_cut = 0;
                for (uint32_t i0 = 0; i0 < na; i0 += kWave) {
                    const uint32_t i = i0 + uint32_t(lane);
                    const uint32_t key = i < na ? h.sorted[i] : 0u;
                    before += wave_sum_u64_of(key > cut.kcut ? weight_of(key) : 0ull);
                    n_cut += uint32_t(__popcll(__ballot(i < na && key == cut.kcut)));
                    if (__ballot(key < cut.kcut) != 0) break;
                }
                const uint64_t w_cut = weight_of(cut.kcut);
                uint64_t r = n_cut;
                if (w_cut > 0) {
                    const uint64_t fit = (theta - before) / w_cut + 1;  // entries t with before + t * w <= theta
                    r = fit < r ? fit : r;
                }
                cut.r_cut = r == n_cut ? 0xffffffffu : uint32_t(r);
                cut.z = before + r * w_cut;
            }
        }
    }
    if (tid == 0) {
        h.cut = cut;
        h.raw_sum = raw_sum;
        h.raw_top = xmax;
        h.ok = ok ? 1u : 0u;
    }
    __syncthreads();
    return (f.use_k || f.use_p) ? ok : true;
}

// Row r of a call (target rows first), and whether it counts: target rows 0 .. len, draft rows 0 .. len - 1.
struct RowRef { int b, j, len; bool target, counts; };
__device__ __forceinline__ RowRef row_ref(const VerifyParams &p, int64_t r) {
    const int64_t n_target = int64_t(p.batch) * (p.k + 1);
    RowRef x;
    x.target = r < n_target;
    const int per = x.target ? p.k + 1 : p.k;
    const int64_t q = x.target ? r : r - n_target;
    x.b = int(q / per);
    x.j = int(q % per);
    x.len = draft_len(p, x.b);
    x.counts = x.target ? x.j <= x.len : x.j < x.len;
    return x;
}

// ---------------------------------------------------------------------------
// fp16 and fp32 rows without top-k, in calls of few rows: the maximum, then the masses (which are 60 instructions an entry: one
// CU takes 50 us for a row of 128,256), by a workgroup per 32 KB of every row.  grid (rows, parts) each; verify_rows goes on from the
// bins.  8 requests x 2 drafts, fp32, top-p 0.9, 128,256 entries: 134 us in verify_rows alone, 6 + 26 + 26
// us so.  What bounds verify_split_mass was not measured: its 60 instructions an entry would take about a third of its time, 64-bit LDS
// atomics on the few bins that hold most entries, and 39 KB of bins cleared and added per 32 KB of the row, are the rest of what it does.
// ---------------------------------------------------------------------------
constexpr int SPLIT_BYTES = 32768;
// Up to how many rows: fp32, top-p 0.9, 128,256 entries, a call of 5 / 40 / 120 / 250 rows: 156 / 165 / 175 / 187 us by a workgroup per
// row, 70 / 95 / 136 / 200 us split; fp16, 50,257 entries: 83 / 105 / 105 / 112 and 67 / 90 / 99 / 124 us.
// (Counted as if every draft had logits: the workspace query does not know.  Looked-up drafts stop being split at little more than half as many rows.)
constexpr int64_t SPLIT_ROWS = 160;
template <typename T> __device__ __forceinline__ int split_span(const VerifyParams &p, int &first) {
    first = int(blockIdx.y) * p.split_entries;
    return p.vocab - first < p.split_entries ? p.vocab - first : p.split_entries;
}
template <typename T> __global__ __launch_bounds__(S_THREADS) void verify_split_top(VerifyParams p) {
    __shared__ uint32_t tops[S_WAVES], bads[S_WAVES];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    if (int(blockIdx.x) >= p.n_rows) return;
    const RowRef x = row_ref(p, blockIdx.x);
    if (!x.counts) return;
    const Filter f = filter_of(p, x.b);
    if (f.use_k) return;
    int first;
    const int count = split_span<T>(p, first);
    uint32_t top = 0, bad = 0;
    each_entry<T>((x.target ? target_row<T>(p, x.b, x.j) : draft_row<T>(p, x.b, x.j)) + first, count, [&](typename T::raw_t raw) {
        const float v = T::widen(raw);
        const uint32_t key = masked_key<T>(v);
        top = key > top && v == v ? key : top;
        bad |= !(v < 256.0f) ? 1u : 0u;
    });
    if (f.use_p)  // the row's bins, for the kernel behind to add to
        for (int i = int(blockIdx.y) * S_THREADS + tid; i < HIST_BINS; i += p.split_parts * S_THREADS)
            p.split_bins[int64_t(blockIdx.x) * HIST_BINS + i] = 0;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const uint32_t o = __shfl_xor(top, off, kWave);
        top = o > top ? o : top;
        bad |= __shfl_xor(bad, off, kWave);
    }
    if (lane == 0) {
        tops[wave] = top;
        bads[wave] = bad;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < S_WAVES; ++w) {
            top = tops[w] > top ? tops[w] : top;
            bad |= bads[w];
        }
        SplitPart &part = p.split[int64_t(blockIdx.x) * p.split_parts + blockIdx.y];
        part.top = top;
        part.bad = bad;
    }
}
template <typename T> __global__ __launch_bounds__(S_THREADS) void verify_split_mass(VerifyParams p) {
    __shared__ uint64_t mass[HIST_BINS];
    __shared__ uint64_t sums[S_WAVES][2];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    if (int(blockIdx.x) >= p.n_rows) return;
    const RowRef x = row_ref(p, blockIdx.x);
    if (!x.counts) return;
    const Filter f = filter_of(p, x.b);
    if (f.use_k) return;
    SplitPart *const parts = p.split + int64_t(blockIdx.x) * p.split_parts;
    uint32_t top, bad;
    split_top(parts, p.split_parts, top, bad);
    if (bad != 0 || top == 0 || !coarse_top(value_of<T>(top))) return;  // (verify_rows sees the same, and takes the radix path)
    if (f.use_p)
        for (int i = tid; i < HIST_BINS; i += S_THREADS) mass[i] = 0;
    __syncthreads();
    int first;
    const int count = split_span<T>(p, first);
    uint64_t all = 0, raw = 0;
    coarse_masses<T>((x.target ? target_row<T>(p, x.b, x.j) : draft_row<T>(p, x.b, x.j)) + first, count, f, x.target && p.out_policy != nullptr,
                     value_of<T>(top), elem_key<T>(raw_of_key<T>(top), f.temp, f.has_t), mass, all, raw);
    all = wave_sum_u64_of(all);
    raw = wave_sum_u64_of(raw);
    if (lane == 0) {
        sums[wave][0] = all;
        sums[wave][1] = raw;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < S_WAVES; ++w) {
            all += sums[w][0];
            raw += sums[w][1];
        }
        parts[blockIdx.y].mass = all;
        parts[blockIdx.y].raw = raw;
    }
    if (f.use_p)
        for (int i = tid; i < HIST_BINS; i += S_THREADS)
            if (mass[i] != 0)
                atomicAdd(reinterpret_cast<unsigned long long *>(&p.split_bins[int64_t(blockIdx.x) * HIST_BINS + i]), (unsigned long long)mass[i]);
}

template <typename T>
__global__ __launch_bounds__(S_THREADS) __attribute__((amdgpu_waves_per_eu(6, 6))) void verify_rows(VerifyParams p) {
    __shared__ VerifyShared<T> lds;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const RowRef ref = row_ref(p, r);
    const bool is_target = ref.target;
    const int b = ref.b, j = ref.j, len = ref.len;
    if (!ref.counts) return;  // the whole workgroup: nobody reads this row's summary
    const typename T::raw_t *rp = is_target ? target_row<T>(p, b, j) : draft_row<T>(p, b, j);
    const bool vec = (is_target ? p.vec_target : p.vec_draft) != 0;
    const Filter f = filter_of(p, b);
    const int64_t d = j < len ? p.draft_ids[int64_t(b) * p.k + j] : -1;
    const bool in_vocab = d >= 0 && d < p.vocab;
    const typename T::raw_t drafted = in_vocab ? rp[d] : typename T::raw_t(0);  // (long before it is needed)
    const bool want_lse = is_target && p.out_policy != nullptr;
    RowCut cut;
    uint32_t raw_cut = 0;
    double raw_sum = 1.0;
    float raw_top = 0.0f;
    bool done = false;
    if constexpr (T::kDtype == KA_DTYPE_BF16) done = hist_cut(lds.row, rp, p.vocab, f, want_lse);
    else done = coarse_cut<T>(lds.row, rp, p.vocab, f, want_lse, p.split_parts > 0 && !f.use_k ? p.split + r * p.split_parts : nullptr,
                              p.split_parts, p.split_bins + r * HIST_BINS);
    if (done) {
        cut = lds.row.cut;
        raw_sum = lds.row.raw_sum;
        raw_top = lds.row.raw_top;
        if constexpr (T::kDtype == KA_DTYPE_BF16) raw_cut = lds.row.raw_cut;
        else if (f.use_k || f.use_p) raw_cut = raw_key_of_cut<T>(cut.kcut, f.temp, f.has_t);
    }
    if (!done) {
        __syncthreads();
        cut = radix_cut<T>(lds.sh, rp, p.vocab, vec, f.temp, f.has_t, f.use_k, f.top_k, f.use_p, f.top_p, true);
        if (f.use_k || f.use_p) raw_cut = raw_key_of_cut<T>(cut.kcut, f.temp, f.has_t);
        if (want_lse) {
            row_lse_to_block<T>(rp, p.vocab, vec, lds.lse);
            __syncthreads();
            if (tid == 0) lds.lse.parts(raw_top, raw_sum);
        }
    }

    // mass of the drafted token; where it sits in a tie group that survives in part, its rank in the group decides
    const uint32_t key = in_vocab ? elem_key<T>(drafted, f.temp, f.has_t) : 0u;
    bool kept = in_vocab && (key > cut.kcut || (key == cut.kcut && key >= cut.kstar));
    if (kept && key == cut.kcut && cut.r_cut != 0xffffffffu) {  // the same for the whole block
        __syncthreads();
        if (tid == 0) lds.ties_before = 0;
        __syncthreads();
        const float low = cut_value<T>(raw_cut);
        uint32_t mine = 0;
        constexpr int U = 8, EPV = T::kPerVec;  // vectors in flight per lane
        for (int64_t base = int64_t(tid) * EPV; base < d; base += U * S_THREADS * EPV) {
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = load_entries<T>(rp, vec, int(d), base + u * S_THREADS * EPV);
#pragma unroll
            for (int u = 0; u < U; ++u)
                mine += uint32_t(__popc(ties_of<T>(v[u], low, base + u * S_THREADS * EPV, int(d), cut.kcut, f)));
        }
        if (mine) atomicAdd(&lds.ties_before, mine);
        __syncthreads();
        kept = lds.ties_before < cut.r_cut;
    }
    if (tid == 0) {
        RowSummary s;
        s.z = cut.z;
        s.w_draft = kept ? weight_fix(key == cut.kmax ? 0.0f : value_of<T>(key) - value_of<T>(cut.kmax)) : 0ull;
        s.raw_sum = raw_sum;
        s.raw_top = raw_top;
        s.pad = 0;
        s.kmax = cut.kmax;
        s.kcut = cut.kcut;
        s.r_cut = cut.r_cut;
        s.raw_cut = raw_cut;
        p.rows[r] = s;
    }
}

// ---------------------------------------------------------------------------
// Residual masses of the stopping position
// ---------------------------------------------------------------------------
constexpr double DRAW_MARGIN = 0x1p-38;

// A row's distribution, entry by entry.
struct RowDist {
    uint32_t kmax, kcut, r_cut;
    int limit;        // entries equal to kcut survive below this index
    float vmax, low;  // unscaled values below `low` have no mass
    uint64_t z;
    double inv;       // 1 / z
    __device__ __forceinline__ bool partial() const { return r_cut != 0xffffffffu; }
    // mass of an entry if the tie group survives; `tie`: it belongs to one that survives in part
    template <typename T> __device__ __forceinline__ uint64_t mass(typename T::raw_t x, const Filter &f, bool &tie) const {
        tie = false;
        if (T::widen(x) < low) return 0ull;
        const uint32_t key = elem_key<T>(x, f.temp, f.has_t);
        if (key < kcut) return 0ull;
        tie = key == kcut && partial();
        return weight_fix(key == kmax ? 0.0f : value_of<T>(key) - vmax);
    }
    template <typename T> __device__ __forceinline__ uint64_t mass_at(typename T::raw_t x, int i, const Filter &f) const {
        bool tie;
        const uint64_t w = mass<T>(x, f, tie);
        return tie && i >= limit ? 0ull : w;
    }
    template <typename T> __device__ __forceinline__ void from(const RowSummary &s) {
        kmax = s.kmax;
        kcut = s.kcut;
        r_cut = s.r_cut;
        limit = 0x7fffffff;
        vmax = value_of<T>(s.kmax);
        low = cut_value<T>(s.raw_cut);
        z = s.z;
        inv = 1.0 / double(s.z);
    }
};

__device__ __forceinline__ double positive(double r) { return r > 0.0 ? r : 0.0; }

// Adds one entry to a share's sums: p and q are its probabilities if the groups survive.
__device__ __forceinline__ void add_entry(ShareSums &s, double p, double q, bool tie_p, bool tie_q) {
    const double r = positive(p - q);
    s.all += r;
    s.without_p += tie_p ? 0.0 : r;
    const double alone = tie_q ? p : r;
    s.without_q += alone;
    s.neither += tie_p ? 0.0 : alone;
    s.ties_p += tie_p ? 1u : 0u;
    s.ties_q += tie_q ? 1u : 0u;
}

// Residual of entry i: max(P - Q, 0); P alone where nothing was rejected, 0 for a looked-up draft that was.
template <typename T> struct Residual {
    const typename T::raw_t *rp, *rq;  // rq null: nothing is subtracted
    bool vec_p, vec_q;
    RowDist p, q;
    int64_t skip;  // the rejected look-up draft, or -1
    Filter f;
    int vocab;

    __device__ __forceinline__ void setup(const VerifyParams &v, int b, int n, int len) {
        f = filter_of(v, b);
        vocab = v.vocab;
        rp = target_row<T>(v, b, n);
        vec_p = v.vec_target != 0;
        p.template from<T>(v.rows[int64_t(b) * (v.k + 1) + n]);
        rq = nullptr;
        vec_q = false;
        skip = -1;
        q = p;
        q.r_cut = 0xffffffffu;
        if (n < len) {
            if (v.draft != nullptr) {
                rq = draft_row<T>(v, b, n);
                vec_q = v.vec_draft != 0;
                q.template from<T>(v.rows[int64_t(v.batch) * (v.k + 1) + int64_t(b) * v.k + n]);
            } else {
                skip = v.draft_ids[int64_t(b) * v.k + n];
            }
        }
    }
    __device__ __forceinline__ uint4 load_p(int64_t base) const { return load_entries<T>(rp, vec_p, vocab, base); }
    __device__ __forceinline__ uint4 load_q(int64_t base) const {
        return rq != nullptr ? load_entries<T>(rq, vec_q, vocab, base) : make_uint4(0, 0, 0, 0);
    }
    // the entries `left` of the vector at `base` into a share's sums
    __device__ __forceinline__ void add_entries(const uint4 &x, const uint4 &y, int64_t base, uint32_t left, ShareSums &s) const {
#pragma unroll 1
        for (; left != 0; left &= left - 1) {
            const int j = __ffs(left) - 1;
            bool tie_p, tie_q = false;
            double pv = double(p.template mass<T>(entry_of<T>(x, j), f, tie_p)) * p.inv;
            if (base + j == skip) pv = 0.0;  // (it still has its place in a tie group)
            const double qv = rq != nullptr ? double(q.template mass<T>(entry_of<T>(y, j), f, tie_q)) * q.inv : 0.0;
            add_entry(s, pv, qv, tie_p, tie_q);
        }
    }
    // each(j, residual) for the entries of the vector at `base` that may have one, in order; the limits are known
    template <typename F> __device__ __forceinline__ void vector(int64_t base, F &&each) const {
        const uint4 x = load_p(base), y = load_q(base);
#pragma unroll 1
        for (uint32_t left = at_least<T>(x, p.low, base, vocab); left != 0; left &= left - 1) {
            const int j = __ffs(left) - 1, i = int(base) + j;
            if (int64_t(i) == skip) continue;
            double r = double(p.template mass_at<T>(entry_of<T>(x, j), i, f)) * p.inv;
            if (rq != nullptr) r -= double(q.template mass_at<T>(entry_of<T>(y, j), i, f)) * q.inv;
            each(j, positive(r));
        }
    }
    // the same in integers, times Z^p Z^q (times Z^p where nothing is subtracted)
    template <typename F> __device__ __forceinline__ void exact_vector(int64_t base, F &&each) const {
        const uint4 x = load_p(base), y = load_q(base);
#pragma unroll 1
        for (uint32_t left = at_least<T>(x, p.low, base, vocab); left != 0; left &= left - 1) {
            const int j = __ffs(left) - 1, i = int(base) + j;
            if (int64_t(i) == skip) continue;
            u128 have = p.template mass_at<T>(entry_of<T>(x, j), i, f), take = 0;
            if (rq != nullptr) {
                have *= q.z;
                take = u128(q.template mass_at<T>(entry_of<T>(y, j), i, f)) * p.z;
            }
            each(j, have > take ? have - take : u128(0));
        }
    }
};

__device__ __forceinline__ u128 shfl_up_of(u128 v, int off) {
    const uint64_t lo = __shfl_up((unsigned long long)uint64_t(v), off, kWave);
    const uint64_t hi = __shfl_up((unsigned long long)uint64_t(v >> 64), off, kWave);
    return (u128(hi) << 64) | lo;
}
__device__ __forceinline__ uint64_t shfl_up_of(uint64_t v, int off) { return __shfl_up((unsigned long long)v, off, kWave); }
__device__ __forceinline__ double shfl_up_of(double v, int off) { return __shfl_up(v, off, kWave); }
template <typename V> __device__ __forceinline__ V wave_incl_scan_of(V v) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const V o = shfl_up_of(v, off);
        if (lane >= off) v += o;
    }
    return v;
}
// Exclusive prefix sum over the block in thread order; `*total` = sum over the block.  Every thread calls it.
template <int WAVES, typename V> __device__ __forceinline__ V block_excl_scan_of(V v, V *wave_buf, V *total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const V inc = wave_incl_scan_of(v);
    __syncthreads();  // wave_buf may still be read from a previous call
    if (lane == kWave - 1) wave_buf[wave] = inc;
    __syncthreads();
    V base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const V x = wave_buf[w];
        if (w < wave) base += x;
        sum += x;
    }
    *total = sum;
    return base + inc - v;
}

// The wavefront's sums over its lanes, in a fixed order; the last lane writes them.  `parts`: some tie group survives in part.
__device__ __forceinline__ void store_share(ShareSums s, bool parts, ShareSums *out) {
    s.all = wave_incl_scan_of(s.all);
    if (parts) {
        s.without_p = wave_incl_scan_of(s.without_p);
        s.without_q = wave_incl_scan_of(s.without_q);
        s.neither = wave_incl_scan_of(s.neither);
        s.ties_p = wave_incl_scan_u32(s.ties_p);
        s.ties_q = wave_incl_scan_u32(s.ties_q);
    }
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) *out = s;
}

// grid (groups of shares, B): a wavefront per share
template <typename T>
__global__ __launch_bounds__(SHARE_THREADS) void verify_shares(VerifyParams p) {
    constexpr int STEPS = SHARE_VECS / kWave;
    const int b = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    const int share = int(blockIdx.x) * (SHARE_THREADS / kWave) + int(threadIdx.x) / kWave;
    const int len = draft_len(p, b);
    const int n = accepted_prefix(p, b, len);
    if (share >= p.n_shares) return;
    Residual<T> res;
    res.setup(p, b, n, len);
    ShareSums sums{};
    uint4 x[STEPS], y[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int64_t base = (int64_t(share) * SHARE_VECS + s * kWave + lane) * T::kPerVec;
        x[s] = res.load_p(base);
        y[s] = res.load_q(base);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int64_t base = (int64_t(share) * SHARE_VECS + s * kWave + lane) * T::kPerVec;
        res.add_entries(x[s], y[s], base, at_least<T>(x[s], res.p.low, base, res.vocab) | (res.q.partial() ? at_least<T>(y[s], res.q.low, base, res.vocab) : 0u), sums);
    }
    store_share(sums, res.p.partial() || res.q.partial(), p.shares + int64_t(b) * p.n_shares + share);
}

// The same for bf16 rows of which many entries survive (no top-k, or a large one): the masses come from two tables in LDS, one
// value per bin of verify_rows, so that an entry costs two reads of LDS instead of two evaluations of the mass polynomial.
// Entries outside the bins (about one in 10^4) are evaluated.  A workgroup builds the tables (9728 evaluations) for
// shares_per_group shares.  grid (groups, B).  64 requests, two rows of 128,256 each (33 MB): 25 us, 1.3 TB/s, a third of it the tables.
constexpr int TABLE_THREADS = 512;
constexpr size_t TABLE_LDS_BYTES = size_t(2) * HIST_BINS * sizeof(double);
__global__ __launch_bounds__(TABLE_THREADS) void verify_shares_table(VerifyParams p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char dyn_lds[];
    double *const tab_p = reinterpret_cast<double *>(dyn_lds), *const tab_q = tab_p + HIST_BINS;
    using T = Bf16;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int len = draft_len(p, b);
    const int n = accepted_prefix(p, b, len);
    Residual<T> res;
    res.setup(p, b, n, len);
    const bool two = res.rq != nullptr, looked_up = res.skip >= 0, parts = res.p.partial() || res.q.partial();
    // a value of a group that survives in part is marked by its sign
    auto probability = [&](const RowDist &d, uint32_t raw) {
        const uint32_t key = elem_key<T>(uint16_t(raw), res.f.temp, res.f.has_t);
        if (key < d.kcut) return 0.0;
        const double v = double(weight_fix(key == d.kmax ? 0.0f : value_of<T>(key) - d.vmax)) * d.inv;
        return d.partial() && key == d.kcut ? -v : v;
    };
#pragma unroll 2
    for (int i = tid; i < HIST_BINS; i += TABLE_THREADS) {
        const uint32_t raw = raw_of_bin(i);
        tab_p[i] = probability(res.p, raw);
        if (two) tab_q[i] = probability(res.q, raw);
    }
    __syncthreads();
    // magnitude bits above the bins' lowest, and the entry's probability where that is below HIST_SIDE
    auto above = [](uint32_t x) { return (x & 0x7fffu) - MAG_LOW; };
    auto value = [](const double *tab, uint32_t m, uint32_t x) { return tab[HIST_SIDE + int(m ^ uint32_t(int32_t(x << 16) >> 31))]; };
    const int first = int(blockIdx.x) * p.shares_per_group;
    const int end = first + p.shares_per_group < p.n_shares ? first + p.shares_per_group : p.n_shares;
    constexpr int STEPS = SHARE_VECS / kWave;
    for (int share = first + wave; share < end; share += TABLE_THREADS / kWave) {
        ShareSums sums{};
        uint4 x[STEPS], y[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int64_t base = (int64_t(share) * SHARE_VECS + s * kWave + lane) * T::kPerVec;
            x[s] = res.load_p(base);
            y[s] = res.load_q(base);
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int64_t base = (int64_t(share) * SHARE_VECS + s * kWave + lane) * T::kPerVec;
            const uint32_t xw[4] = {x[s].x, x[s].y, x[s].z, x[s].w}, yw[4] = {y[s].x, y[s].y, y[s].z, y[s].w};
            if (base >= res.vocab) continue;
            // entries evaluated one by one: outside the bins, and all of the row's last vector if it is cut short
            const bool whole = base + 8 <= res.vocab;
            uint32_t odd = whole ? 0u : (1u << int(res.vocab - base)) - 1u;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t xe = xw[j / 2] >> (16 * (j & 1)), ye = yw[j / 2] >> (16 * (j & 1));
                const uint32_t mx = above(xe), my = above(ye);
                if (mx >= uint32_t(HIST_SIDE) || (two && my >= uint32_t(HIST_SIDE))) {
                    odd |= whole ? 1u << j : 0u;
                } else if (whole) {
                    const double pv = value(tab_p, mx, xe), qv = two ? value(tab_q, my, ye) : 0.0;
                    const bool skipped = looked_up && base + j == res.skip;
                    if (!parts) sums.all += skipped ? 0.0 : positive(pv - qv);
                    else add_entry(sums, skipped ? 0.0 : fabs(pv), fabs(qv), pv < 0.0, qv < 0.0);
                }
            }
            res.add_entries(x[s], y[s], base, odd, sums);
        }
        store_share(sums, parts, p.shares + int64_t(b) * p.n_shares + share);
    }
}

// The draw in integers, by the whole block (blocks of SHARE_VECS threads): the total, then the entry.
template <typename T> __device__ __forceinline__ int exact_draw(Residual<T> res, float u, int n_shares, u128 *wave_buf, int *hit) {
    constexpr int WAVES = SHARE_VECS / kWave;
    const int tid = threadIdx.x;
    u128 tau = 0;
    for (int turn = 0; turn < 2; ++turn) {
        u128 at = 0;
        for (int share = 0; share < n_shares; ++share) {  // block-uniform: `at` and the totals are
            const int64_t base = (int64_t(share) * SHARE_VECS + tid) * T::kPerVec;
            u128 sum = 0, total;
            res.exact_vector(base, [&](int, u128 m) { sum += m; });
            u128 before = at + block_excl_scan_of<WAVES, u128>(sum, wave_buf, &total);
            at += total;
            if (turn == 0) continue;
            if (before <= tau && tau < before + sum) {
                int found = -1;
                res.exact_vector(base, [&](int j, u128 m) {
                    before += m;
                    if (found < 0 && tau < before) found = int(base) + j;
                });
                *hit = found;
            }
            if (tau < at) break;
        }
        if (turn == 0) {
            if (at == 0) {  // no residual (see the head of the file): drawn from P
                res.rq = nullptr;
                res.skip = -1;
                at = res.p.z;
            }
            tau = floor_scale_wide(u, at);
        }
    }
    __syncthreads();
    return *hit;
}

// grid B; a thread per vector of the share that holds the draw
// verify_draw: grid (B).  Bound by its chain of waits, not by what it reads: the request's summaries, its shares, two vectors; 8 us for one
// request, 11 for 64, 13.5 where top-p cuts inside tie groups, 16 for 256.
template <typename T>
__global__ __launch_bounds__(SHARE_VECS) void verify_draw(VerifyParams p) {
    constexpr int WAVES = SHARE_VECS / kWave, EPV = T::kPerVec;
    __shared__ union { double d[WAVES]; uint64_t u[WAVES]; u128 w[WAVES]; } wave_buf;
    __shared__ double s_before, s_value[2];
    __shared__ int s_share, s_hit, s_cut[2], s_limit[2];
    __shared__ uint32_t s_rank[2];
    const int b = blockIdx.x, tid = threadIdx.x;
    const int len = draft_len(p, b);
    // thread t takes a run of shares, as a rule one; it is requested ahead of the positions' decision
    const ShareSums *const shares = p.shares + int64_t(b) * p.n_shares;
    const int per = (p.n_shares + SHARE_VECS - 1) / SHARE_VECS;
    const int s0 = tid * per, s1 = s0 + per < p.n_shares ? s0 + per : p.n_shares;
    const ShareSums first = shares[s0 < p.n_shares ? s0 : 0];
    auto share_at = [&](int s) { return s == s0 ? first : shares[s]; };
    // what thread j needs for its output at position j, ahead of the draw: the draft, its logit and the row's log-sum-exp
    const bool has_row = tid <= len, has_draft = tid < len;
    const int64_t drafted = has_draft ? p.draft_ids[int64_t(b) * p.k + tid] : -1;
    double lse = 0.0;
    float logit = 0.0f;
    if (p.out_policy != nullptr && has_row) {
        const RowSummary &row = p.rows[int64_t(b) * (p.k + 1) + tid];
        if (drafted >= 0 && drafted < p.vocab) logit = T::widen(target_row<T>(p, b, tid)[drafted]);
        lse = double(row.raw_top) + log(row.raw_sum);
    }
    const int n = accepted_prefix(p, b, len);
    if (tid == 0) { s_share = s_hit = -1; s_cut[0] = s_cut[1] = -1; s_limit[0] = s_limit[1] = 0x7fffffff; }
    const float u = clean_uniform(p.uniforms[int64_t(b) * (p.k + 1) + p.k]);
    Residual<T> res;
    res.setup(p, b, n, len);
    const bool parts = res.p.partial() || res.q.partial();
    uint32_t before_p = 0, before_q = 0;  // ties in front of the thread's shares
    if (parts) {
        // ---- the shares and the indices at which the groups are cut ----
        uint32_t cp = 0, cq = 0;
        for (int s = s0; s < s1; ++s) { cp += share_at(s).ties_p; cq += share_at(s).ties_q; }
        uint64_t total;
        const uint64_t both = block_excl_scan_of<WAVES, uint64_t>((uint64_t(cq) << 32) | cp, wave_buf.u, &total);
        before_p = uint32_t(both);
        before_q = uint32_t(both >> 32);
        uint32_t rp = before_p, rq = before_q;
        for (int s = s0; s < s1; ++s) {
            const uint32_t ties_p = share_at(s).ties_p, ties_q = share_at(s).ties_q;
            // the share that holds the last survivor, and how many of its entries survive
            if (res.p.partial() && rp < res.p.r_cut && res.p.r_cut <= rp + ties_p) { s_cut[0] = s; s_rank[0] = res.p.r_cut - rp; }
            if (res.q.partial() && rq < res.q.r_cut && res.q.r_cut <= rq + ties_q) { s_cut[1] = s; s_rank[1] = res.q.r_cut - rq; }
            rp += ties_p;
            rq += ties_q;
        }
        __syncthreads();
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            const RowDist &d = side == 0 ? res.p : res.q;
            if (!d.partial() || s_cut[side] < 0) continue;  // block-uniform
            const int64_t base = (int64_t(s_cut[side]) * SHARE_VECS + tid) * EPV;
            uint32_t group = ties_of<T>(side == 0 ? res.load_p(base) : res.load_q(base), d.low, base, p.vocab, d.kcut, res.f);
            uint64_t all;
            const uint32_t rank = uint32_t(block_excl_scan_of<WAVES, uint64_t>(uint64_t(__popc(group)), wave_buf.u, &all));
            if (rank < s_rank[side] && s_rank[side] <= rank + uint32_t(__popc(group))) {
                for (uint32_t skip = s_rank[side] - rank - 1; skip != 0; --skip) group &= group - 1;
                s_limit[side] = int(base) + __ffs(group);  // the last survivor's index + 1
            }
        }
        __syncthreads();
        res.p.limit = s_limit[0];
        res.q.limit = s_limit[1];
        // ---- the one or two shares that are cut, with the limits known ----
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            if (s_cut[side] < 0 || (side == 1 && s_cut[1] == s_cut[0])) continue;
            double sum = 0.0, total_here;
            res.vector((int64_t(s_cut[side]) * SHARE_VECS + tid) * EPV, [&](int, double r) { sum += r; });
            block_excl_scan_of<WAVES, double>(sum, wave_buf.d, &total_here);
            if (tid == 0) s_value[side] = total_here;
        }
        __syncthreads();
    }
    // a share's sum, given the ties in front of it
    auto share_sum = [&](int s, uint32_t &rp, uint32_t &rq) {
        const ShareSums x = share_at(s);
        if (!parts) return x.all;
        const bool out_p = res.p.partial() && rp >= res.p.r_cut, out_q = res.q.partial() && rq >= res.q.r_cut;
        rp += x.ties_p;
        rq += x.ties_q;
        if (s == s_cut[0]) return s_value[0];
        if (s == s_cut[1]) return s_value[1];
        return out_p ? (out_q ? x.neither : x.without_p) : (out_q ? x.without_q : x.all);
    };
    // the share that holds u R
    double mine = 0.0, r;
    {
        uint32_t rp = before_p, rq = before_q;
        for (int s = s0; s < s1; ++s) mine += share_sum(s, rp, rq);
    }
    const double excl = block_excl_scan_of<WAVES, double>(mine, wave_buf.d, &r);
    const double tau = double(u) * r;
    if (excl <= tau && tau < excl + mine) {
        double at = excl;
        uint32_t rp = before_p, rq = before_q;
        for (int s = s0; s < s1; ++s) {
            const double m = share_sum(s, rp, rq);
            // (near a border two threads can take tau for theirs: neither keeps the margin then)
            if (tau - at >= DRAW_MARGIN && at + m - tau >= DRAW_MARGIN) { s_share = s; s_before = at; break; }
            at += m;
        }
    }
    __syncthreads();
    if (s_share >= 0) {  // the same for the whole block
        const int64_t base = (int64_t(s_share) * SHARE_VECS + tid) * EPV;
        double m[EPV], sum = 0.0, total;
#pragma unroll
        for (int j = 0; j < EPV; ++j) m[j] = 0.0;
        res.vector(base, [&](int j, double v) {
#pragma unroll
            for (int k = 0; k < EPV; ++k) m[k] = j == k ? v : m[k];
            sum += v;
        });
        double before = s_before + block_excl_scan_of<WAVES, double>(sum, wave_buf.d, &total);
        if (before <= tau && tau < before + sum) {
            bool found = false;
#pragma unroll
            for (int j = 0; j < EPV; ++j) {
                if (!found && tau < before + m[j]) {
                    found = true;
                    if (tau - before >= DRAW_MARGIN && before + m[j] - tau >= DRAW_MARGIN) s_hit = int(base) + j;
                }
                before += m[j];
            }
        }
    }
    __syncthreads();
    int hit = s_hit;
    if (hit < 0) {  // block-uniform
        __syncthreads();
        hit = exact_draw<T>(res, u, p.n_shares, wave_buf.w, &s_hit);
    }
    // outputs: thread j writes position j
    if (tid <= p.k) {
        const int64_t at = int64_t(b) * (p.k + 1) + tid;
        const int64_t id = tid < n ? drafted : (tid == n ? int64_t(hit) : int64_t(-1));
        p.out_ids[at] = id;
        if (p.out_policy != nullptr) {
            float lp = 0.0f;
            if (tid <= n) {
                if (tid == n && id >= 0) logit = T::widen(target_row<T>(p, b, tid)[id]);
                lp = id >= 0 ? float(double(logit) - lse) : __builtin_nanf("");
            }
            p.out_policy[at] = lp;
        }
    }
    if (tid == 0) p.out_accepted[b] = n;
}

// verify_shares_table uses 78 KB of LDS: the attribute belongs to the device, set once for each (or twice, by two threads at once).
inline int reserve_table_lds() {
    static std::atomic<bool> done[64];
    int device = 0;
    hipError_t rc = hipGetDevice(&device);
    if (rc != hipSuccess) return check_hip(rc, "verify: hipGetDevice");
    if (device < 0 || device >= 64) return fail(KA_ERR_UNSUPPORTED, "verify: device index %d", device);
    if (!done[device].load(std::memory_order_acquire)) {
        rc = hipFuncSetAttribute(reinterpret_cast<const void *>(verify_shares_table), hipFuncAttributeMaxDynamicSharedMemorySize, int(TABLE_LDS_BYTES));
        if (rc != hipSuccess) return check_hip(rc, "verify: reserving LDS for the tables");
        done[device].store(true, std::memory_order_release);
    }
    return KA_OK;
}

template <typename T> int launch_verify(const VerifyParams &p, hipStream_t stream) {
    const int64_t rows = int64_t(p.batch) * (p.k + 1) + (p.draft != nullptr ? int64_t(p.batch) * p.k : 0);
    int rc = KA_OK;
    if constexpr (T::kDtype != KA_DTYPE_BF16) {
        if (p.split_parts > 0) {
            const dim3 grid{unsigned((rows + 7) / 8 * 8), unsigned(p.split_parts)};  // all parts of a row on one XCD
            hipLaunchKernelGGL((verify_split_top<T>), grid, dim3(S_THREADS), 0, stream, p);
            rc = check_hip(hipGetLastError(), "verify launch (maxima)");
            if (rc != KA_OK) return rc;
            hipLaunchKernelGGL((verify_split_mass<T>), grid, dim3(S_THREADS), 0, stream, p);
            rc = check_hip(hipGetLastError(), "verify launch (masses)");
            if (rc != KA_OK) return rc;
        }
    }
    hipLaunchKernelGGL((verify_rows<T>), dim3(unsigned(rows)), dim3(S_THREADS), 0, stream, p);
    rc = check_hip(hipGetLastError(), "verify launch (rows)");
    if (rc != KA_OK) return rc;
    if (T::kDtype == KA_DTYPE_BF16 && p.shares_per_group > 0) {
        rc = reserve_table_lds();
        if (rc != KA_OK) return rc;
        hipLaunchKernelGGL(verify_shares_table, dim3(unsigned((p.n_shares + p.shares_per_group - 1) / p.shares_per_group), unsigned(p.batch)),
                           dim3(TABLE_THREADS), TABLE_LDS_BYTES, stream, p);
    } else {
        hipLaunchKernelGGL((verify_shares<T>), dim3(unsigned((p.n_shares * kWave + SHARE_THREADS - 1) / SHARE_THREADS), unsigned(p.batch)), dim3(SHARE_THREADS), 0, stream, p);
    }
    rc = check_hip(hipGetLastError(), "verify launch (shares)");
    if (rc != KA_OK) return rc;
    hipLaunchKernelGGL((verify_draw<T>), dim3(unsigned(p.batch)), dim3(SHARE_VECS), 0, stream, p);
    return check_hip(hipGetLastError(), "verify launch (draw)");
}

inline size_t align_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

struct VerifyLayout {
    int64_t n_shares, split_parts;
    size_t rows, shares, split, split_bins, total;
};
inline VerifyLayout verify_layout(int dtype, int64_t batch, int64_t k, int64_t vocab) {
    VerifyLayout l;
    const int64_t epv = dtype == KA_DTYPE_F32 ? 4 : 8;
    l.n_shares = (vocab + SHARE_VECS * epv - 1) / (SHARE_VECS * epv);
    l.rows = 0;
    l.shares = align_up(size_t(batch) * size_t(2 * k + 1) * sizeof(RowSummary), 256);
    l.total = l.shares + size_t(batch) * size_t(l.n_shares) * sizeof(ShareSums);
    l.split = align_up(l.total, 256);
    const int64_t n_rows = batch * (2 * k + 1), parts = (vocab + SPLIT_BYTES / (16 / epv) - 1) / (SPLIT_BYTES / (16 / epv));
    l.split_parts = dtype != KA_DTYPE_BF16 && parts > 1 && n_rows <= SPLIT_ROWS ? parts : 0;
    l.split_bins = align_up(l.split + size_t(n_rows) * size_t(l.split_parts) * sizeof(SplitPart), 256);
    if (l.split_parts > 0) l.total = l.split_bins + size_t(n_rows) * HIST_BINS * sizeof(uint64_t);
    return l;
}

}  // namespace
}  // namespace ka

KA_EXPORT size_t ka_verify_workspace_bytes(int dtype, int64_t batch, int64_t max_draft, int64_t vocab) {
    if ((dtype != KA_DTYPE_BF16 && dtype != KA_DTYPE_F16 && dtype != KA_DTYPE_F32) || batch <= 0 || max_draft < 0 ||
        max_draft > ka::VERIFY_MAX_DRAFT || vocab < 1 || vocab >= ka::VERIFY_MAX_VOCAB || batch > ka::VERIFY_MAX_BATCH ||
        batch * (2 * max_draft + 1) >= ka::VERIFY_MAX_ROWS)
        return 0;
    return ka::verify_layout(dtype, batch, max_draft, vocab).total;
}

KA_EXPORT int ka_verify_draft(int dtype, const void *target_logits, int64_t target_batch_stride, int64_t target_pos_stride,
                              const void *draft_logits, int64_t draft_batch_stride, int64_t draft_pos_stride,
                              const int64_t *draft_ids, const int64_t *draft_lens, const float *uniforms, int64_t batch,
                              int64_t max_draft, int64_t vocab, float temperature, const float *temperature_rows,
                              int32_t top_k, const int32_t *top_k_rows, float top_p, const float *top_p_rows,
                              int64_t *out_ids, int64_t *out_accepted, float *out_policy_logprob, void *workspace,
                              size_t workspace_bytes, void *hip_stream) {
    using namespace ka;
    if (dtype != KA_DTYPE_BF16 && dtype != KA_DTYPE_F16 && dtype != KA_DTYPE_F32)
        return fail(KA_ERR_BAD_ARG, "verify: unknown dtype code %d", dtype);
    if (batch < 0) return fail(KA_ERR_BAD_ARG, "verify: batch %lld < 0", (long long)batch);
    if (max_draft < 0) return fail(KA_ERR_BAD_ARG, "verify: max_draft %lld < 0", (long long)max_draft);
    if (max_draft > VERIFY_MAX_DRAFT)
        return fail(KA_ERR_UNSUPPORTED, "verify: max_draft %lld > %d", (long long)max_draft, VERIFY_MAX_DRAFT);
    if (batch == 0) return KA_OK;
    if (target_logits == nullptr || uniforms == nullptr || out_ids == nullptr || out_accepted == nullptr ||
        (draft_ids == nullptr && max_draft > 0))
        return fail(KA_ERR_BAD_ARG, "verify: null target_logits / draft_ids / uniforms / out_ids / out_accepted pointer");
    if (vocab < 1) return fail(KA_ERR_BAD_ARG, "verify: vocab %lld < 1", (long long)vocab);
    if (vocab >= VERIFY_MAX_VOCAB)
        return fail(KA_ERR_UNSUPPORTED, "verify: vocab %lld >= 2^22 (integer masses would overflow)", (long long)vocab);
    if (batch > VERIFY_MAX_BATCH) return fail(KA_ERR_UNSUPPORTED, "verify: batch %lld > %lld", (long long)batch, (long long)VERIFY_MAX_BATCH);
    if (batch * (2 * max_draft + 1) >= VERIFY_MAX_ROWS)
        return fail(KA_ERR_UNSUPPORTED, "verify: %lld rows in one call", (long long)(batch * (2 * max_draft + 1)));
    // (a stride counts only where there is a second row to step to)
    if ((batch > 1 && target_batch_stride < vocab) || (max_draft > 0 && target_pos_stride < vocab))
        return fail(KA_ERR_BAD_ARG, "verify: a target stride is smaller than the vocabulary");
    if (draft_logits != nullptr && ((batch > 1 && max_draft > 0 && draft_batch_stride < vocab) || (max_draft > 1 && draft_pos_stride < vocab)))
        return fail(KA_ERR_BAD_ARG, "verify: a draft stride is smaller than the vocabulary");
    if (temperature_rows == nullptr && !(temperature > 0.0f))
        return fail(KA_ERR_BAD_ARG, "verify: temperature %g must be > 0", temperature);
    if (top_k_rows == nullptr && top_k < 0) return fail(KA_ERR_BAD_ARG, "verify: top_k %d < 0", top_k);
    if (top_p_rows == nullptr && !(top_p > 0.0f && top_p <= 1.0f))
        return fail(KA_ERR_BAD_ARG, "verify: top_p %g outside (0, 1]", top_p);
    const VerifyLayout l = verify_layout(dtype, batch, max_draft, vocab);
    if (workspace == nullptr || workspace_bytes < l.total)
        return fail(KA_ERR_WORKSPACE, "verify: workspace of %zu B, need %zu B", workspace == nullptr ? size_t(0) : workspace_bytes, l.total);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(KA_ERR_BAD_ARG, "verify: workspace is not 16-byte aligned");
    const int64_t esize = dtype == KA_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(target_logits) % size_t(esize) != 0 || reinterpret_cast<uintptr_t>(draft_logits) % size_t(esize) != 0)
        return fail(KA_ERR_BAD_ARG, "verify: logits are not aligned to their element");
    VerifyParams p{};
    p.target = target_logits;
    p.draft = max_draft > 0 ? draft_logits : nullptr;
    p.t_batch = target_batch_stride;
    p.t_pos = target_pos_stride;
    p.d_batch = draft_batch_stride;
    p.d_pos = draft_pos_stride;
    p.draft_ids = draft_ids;
    p.draft_lens = draft_lens;
    p.uniforms = uniforms;
    p.batch = int32_t(batch);
    p.k = int32_t(max_draft);
    p.vocab = int32_t(vocab);
    p.temperature = temperature;
    p.temperature_rows = temperature_rows;
    p.top_k = top_k;
    p.top_k_rows = top_k_rows;
    p.top_p = top_p;
    p.top_p_rows = top_p_rows;
    p.out_ids = out_ids;
    p.out_accepted = out_accepted;
    p.out_policy = out_policy_logprob;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    p.rows = reinterpret_cast<RowSummary *>(ws + l.rows);
    p.shares = reinterpret_cast<ShareSums *>(ws + l.shares);
    p.n_shares = int32_t(l.n_shares);
    if (l.split_parts > 0 && (top_k_rows != nullptr || top_k == 0 || top_k >= vocab)) {
        p.n_rows = int32_t(batch * (max_draft + 1) + (p.draft != nullptr ? batch * max_draft : 0));
        p.split_parts = int32_t(l.split_parts);
        p.split_entries = int32_t(SPLIT_BYTES / esize);
        p.split = reinterpret_cast<SplitPart *>(ws + l.split);
        p.split_bins = reinterpret_cast<uint64_t *>(ws + l.split_bins);
    }
    // Tables pay where most entries may have mass: two of them cost 9728 evaluations, a share of 2048 entries 4096 without.  64 requests x
    // 4 drafts, us a call with tables and without: no filter, 128,256 / 32,768 / 8192 entries: 91 / 114, 55 / 61, 48 / 54; top-p 0.9,
    // 128,256 / 22,000 / 8192: 96 / 98, 61 / 59, 60 / 56; top-k 50: 71 / 64.
    // Enough groups to fill the device twice, of at least eight shares (one per wavefront).
    const bool many = top_k_rows != nullptr || top_k == 0 || top_k > 1024;
    const bool whole = top_k_rows == nullptr && top_k == 0 && top_p_rows == nullptr && top_p >= 1.0f;
    if (dtype == KA_DTYPE_BF16 && many && l.n_shares >= (whole ? 4 : 16)) {
        int64_t groups = (512 + batch - 1) / batch;
        if (groups > (l.n_shares + 7) / 8) groups = (l.n_shares + 7) / 8;
        p.shares_per_group = int32_t(((l.n_shares + groups - 1) / groups + 7) / 8 * 8);
    }
    auto aligned = [&](const void *base, int64_t batch_stride, int64_t pos_stride, int64_t positions) {
        return reinterpret_cast<uintptr_t>(base) % 16 == 0 && (batch == 1 || (batch_stride * esize) % 16 == 0) &&
               (positions <= 1 || (pos_stride * esize) % 16 == 0);
    };
    p.vec_target = aligned(target_logits, target_batch_stride, target_pos_stride, max_draft + 1) ? 1 : 0;
    p.vec_draft = p.draft != nullptr && aligned(draft_logits, draft_batch_stride, draft_pos_stride, max_draft) ? 1 : 0;
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    if (dtype == KA_DTYPE_BF16) return launch_verify<Bf16>(p, stream);
    if (dtype == KA_DTYPE_F16) return launch_verify<F16>(p, stream);
    return launch_verify<F32>(p, stream);
}
