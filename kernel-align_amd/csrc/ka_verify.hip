// Verification of drafted tokens: a drafter proposes up to K tokens per request, the target model scores the K + 1 positions
// in one forward pass, and the tokens are accepted or redrawn so that what comes out is distributed as the sampling operator
// would draw it from the target rows alone (speculative sampling).
//
//   P = W^p / Z^p, Q = W^q / Z^q      the rows' distributions after temperature, top-k and top-p, as integer masses: those of
//                                     the sampling kernels (Q is one-hot at the draft when there are no draft logits)
//   position j accepts d_j  iff  u_j Q(d_j) < P(d_j);  n = the first position that does not, or the number of drafts
//   ids[n] = inverse CDF, in index order, of max(P - Q, 0) (rejected) or of P (every draft accepted)
//
// Everything is decided on integers: u_j W^q Z^p < W^p Z^q (126 bits), residual masses max(W^p Z^q - W^q Z^p, 0) (102 bits
// each, 124 bits in sum).  A rejected draft with Q(d) > 0 always leaves a residual: P(d) <= u Q(d) < Q(d), both sum to one
// exactly, so some other entry has P > Q.  A draft that Q cannot have drawn (filtered out, or no entry at all) may meet P = Q:
// then the token is drawn from P.  Nothing depends on the order of a sum, on the batch or on the launch.
//
// Four launches, no host synchronisation:
//   verify_rows    one workgroup per row that counts (target rows 0 .. len, draft rows 0 .. len - 1): the cut of the row's
//                  distribution, its total mass, the draft token's mass, the log-sum-exp of the raw row.  This is the pass over
//                  the data: bound by HBM, 2 V (2 K + 1) bytes per request.
//   verify_ties    (only where top-p may cut inside a group of equal logits) the index at which the cut falls, for the two rows
//                  of the position where the request stops
//   verify_shares  residual mass of every share of 256 vectors of the stopping position, a wavefront each
//   verify_draw    one workgroup per request: the share, the vector and the entry that hold the draw; all outputs
// The rows of the stopping position are read again by the last two, from L2 / MALL as a rule.
#define KA_SAMPLING_THREADS 512
#include <stddef.h>

#include "ka_sampling_common.h"
#include "ka_sampling_radix.h"

namespace ka {
namespace {

typedef unsigned __int128 u128;

constexpr int VERIFY_MAX_DRAFT = KA_VERIFY_MAX_DRAFT;
static_assert(VERIFY_MAX_DRAFT <= kWave, "one lane decides one position");
constexpr int SHARE_VECS = 256;    // 16-byte vectors of a row in one share; verify_draw has a thread for each
constexpr int SHARE_THREADS = 256;

// What verify_rows leaves about a row.
struct RowSummary {
    uint64_t z;         // integer mass of the survivors
    uint64_t w_draft;   // of which the drafted token has this (0: filtered out, or an id outside the vocabulary)
    double lse;         // log-sum-exp of the raw row (target rows, when asked for)
    uint32_t kmax, kcut, r_cut;  // see RowCut
    uint32_t raw_cut;   // key (unscaled) below which no entry survives; 0: not known, or no filter
};
static_assert(sizeof(RowSummary) == 40, "the workspace query counts 40 bytes per row");

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
    int32_t *tie_limit;                                  // [B, 2]: an entry equal to kcut survives iff its index is below this
    u128 *shares;                                        // [B, n_shares]
    int32_t n_shares, vec_target, vec_draft, may_cut_ties;
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
__device__ __forceinline__ void load_entries(const typename T::raw_t *row, bool vec, int vocab, int64_t base, typename T::raw_t (&e)[T::kPerVec]) {
    constexpr int EPV = T::kPerVec;
    if (vec && base + EPV <= vocab) {
        const uint4 v = *reinterpret_cast<const uint4 *>(row + base);
        __builtin_memcpy(e, &v, 16);
    } else {
#pragma unroll
        for (int j = 0; j < EPV; ++j) e[j] = base + j < vocab ? row[base + j] : typename T::raw_t(0);
    }
}
// The value below which an unscaled entry does not survive (NaN compares as surviving: its key decides).
template <typename T> __device__ __forceinline__ float cut_value(uint32_t raw_cut) {
    return raw_cut == 0 ? -__builtin_inff() : value_of<T>(raw_cut);
}

// ---------------------------------------------------------------------------
// verify_rows
//
// A bf16 row has few distinct values, and everything a summary holds is a function of how often each occurs: one streaming
// pass counts the values of 2^-7 <= |x| < 2^8 in 3840 bins (15 KB of LDS, so that three workgroups share a CU and one row's
// tail runs under the reads of the others), lists the few smaller ones, and drops x <= -2^8, which has no mass next to an
// ordinary maximum.  The masses are then evaluated once per occupied bin instead of once per entry, and a scan over the bins
// in descending order finds the cuts.  Rows it cannot describe (values of 2^8 and above, NaN, a maximum or a cut among the
// small values, dropped values that would count) take the radix path, as fp16 and fp32 rows do.
// ---------------------------------------------------------------------------
constexpr int HIST_SIDE = 15 * 128;          // values of one sign: 15 octaves of 128
constexpr int HIST_BINS = 2 * HIST_SIDE;     // ascending: negative values first
constexpr int HIST_POS = HIST_BINS + 1;      // positions in descending order: positive bins, the small values, negative bins
constexpr int HIST_PER = (HIST_POS + S_THREADS - 1) / S_THREADS;
constexpr uint32_t MAG_LOW = 0x3C00u, MAG_HIGH = 0x4380u;  // bits of 2^-7 and 2^8
constexpr int TINY_CAP = 2048;
static_assert(MAG_HIGH - MAG_LOW == uint32_t(HIST_SIDE), "the bins cover [2^-7, 2^8)");

struct HistRow {
    uint32_t bin[HIST_BINS];
    uint16_t tiny[TINY_CAP];
    uint32_t n_tiny, n_zero, give_up, dropped;
    uint32_t first, kpos, kstar, best, kcut, n_cut, last;
    unsigned long long before;
    uint64_t wave_u64[S_WAVES];
    uint32_t wave_u32[S_WAVES];
};
struct VerifyShared {
    union {
        Shared sh;
        HistRow hist;
    };
    PolicyLse lse;
    uint32_t ties_before;
};

__device__ __forceinline__ uint32_t raw_of_bin(int bin) {
    return bin >= HIST_SIDE ? MAG_LOW + uint32_t(bin - HIST_SIDE) : 0x8000u | (MAG_LOW + uint32_t(HIST_SIDE - 1 - bin));
}
__device__ __forceinline__ int bin_of_pos(int q) { return q < HIST_SIDE ? HIST_BINS - 1 - q : HIST_BINS - q; }

// False: the row needs the radix path (nothing is decided).  Every thread gets the results; *lse only with want_lse.
__device__ __forceinline__ bool hist_cut(HistRow &h, const uint16_t *rp, int vocab, const Filter &f, bool want_lse, RowCut &cut,
                                         uint32_t &raw_cut, double &lse) {
    const int tid = threadIdx.x;
    for (int i = tid; i < HIST_BINS; i += S_THREADS) h.bin[i] = 0;
    if (tid == 0) { h.n_tiny = h.n_zero = h.give_up = h.dropped = 0; h.best = h.last = 0; h.n_cut = 0; h.before = ~0ull; }
    __syncthreads();
    // ---- one pass over the row -------------------------------------------------------------
    {
        uint32_t zeros = 0, high = 0, low = 0;
        auto odd = [&](uint32_t x) {  // |x| outside the bins
            const uint32_t mag = x & 0x7fffu;
            if (mag == 0) ++zeros;
            else if (mag < MAG_LOW) {
                const uint32_t at = atomicAdd(&h.n_tiny, 1u);
                if (at < uint32_t(TINY_CAP)) h.tiny[at] = uint16_t(x);
            } else if ((x & 0x8000u) == 0 || mag > 0x7f80u) high = 1;
            else low = 1;
        };
        auto count = [&](uint32_t x) {
            const uint32_t m = (x & 0x7fffu) - MAG_LOW, sign = uint32_t(int32_t(x << 16) >> 31);
            if (m < uint32_t(HIST_SIDE)) atomicAdd(&h.bin[HIST_SIDE + int(m ^ sign)], 1u);
            else odd(x & 0xffffu);
        };
        auto count_vector = [&](const uint4 &q) {
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                count(w[j]);
                count(w[j] >> 16);
            }
        };
        int head = int((16 - (reinterpret_cast<uintptr_t>(rp) & 15)) & 15) / 2;  // entries before the first whole vector
        head = head < vocab ? head : vocab;
        if (tid < head) count(rp[tid]);
        const uint4 *vp = reinterpret_cast<const uint4 *>(rp + head);
        const int nvec = (vocab - head) / 8;
        constexpr int U = 8;  // loads in flight per lane
        int v = tid;
        for (; v + (U - 1) * S_THREADS < nvec; v += U * S_THREADS) {
            uint4 q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = load_stream(vp + v + u * S_THREADS);
#pragma unroll
            for (int u = 0; u < U; ++u) count_vector(q[u]);
        }
        for (; v < nvec; v += S_THREADS) count_vector(load_stream(vp + v));
        const int i = head + nvec * 8 + tid;
        if (i < vocab) count(rp[i]);
        if (zeros) atomicAdd(&h.n_zero, zeros);
        if (high) h.give_up = 1;
        if (low) h.dropped = 1;
    }
    __syncthreads();
    const uint32_t n_tiny = h.n_tiny, n_zero = h.n_zero, dropped = h.dropped;
    if (h.give_up != 0 || n_tiny > uint32_t(TINY_CAP)) return false;
    const uint32_t n_mid = n_tiny + n_zero;
    auto key_of_raw = [&](uint32_t raw) { return elem_key<Bf16>(uint16_t(raw), f.temp, f.has_t); };

    // ---- the thread's positions ------------------------------------------------------------
    uint32_t c[HIST_PER], sk[HIST_PER], mine = 0;
#pragma unroll
    for (int j = 0; j < HIST_PER; ++j) {
        const int q = tid * HIST_PER + j;
        c[j] = q >= HIST_POS ? 0u : (q == HIST_SIDE ? n_mid : h.bin[bin_of_pos(q)]);
        mine += c[j];
    }
    uint32_t counted;
    const uint32_t rank0 = block_excl_scan<uint32_t>(mine, h.wave_u32, &counted);
    if (counted == 0) return false;
    if (rank0 == 0 && mine > 0) {
        int j = 0;
        while (c[j] == 0) ++j;
        h.first = uint32_t(tid * HIST_PER + j);
    }
    if (f.use_k && rank0 < uint32_t(f.top_k) && uint32_t(f.top_k) <= rank0 + mine) {
        uint32_t run = rank0;
        int at = 0;
#pragma unroll
        for (int j = 0; j < HIST_PER; ++j) {
            if (run < uint32_t(f.top_k) && uint32_t(f.top_k) <= run + c[j]) at = j;
            run += c[j];
        }
        const int q = tid * HIST_PER + at;
        h.kpos = uint32_t(q);
        h.kstar = q == HIST_SIDE ? 0u : key_of_raw(raw_of_bin(bin_of_pos(q)));
    }
    __syncthreads();
    const int first = int(h.first);
    if (first == HIST_SIDE || (f.use_k && (counted < uint32_t(f.top_k) || h.kpos == uint32_t(HIST_SIDE)))) return false;
    const uint32_t raw_max = raw_of_bin(bin_of_pos(first));
    const uint32_t kmax = key_of_raw(raw_max);
    const float vmax = value_of<Bf16>(kmax), xmax = Bf16::widen(uint16_t(raw_max));
    const uint32_t kstar = f.use_k ? h.kstar : 0u;
    const uint32_t key_dropped = key_of_raw(0x8000u | MAG_HIGH), key_tiny = key_of_raw(MAG_LOW - 1), key_tiny_neg = key_of_raw(0x8000u | (MAG_LOW - 1));
    if (dropped && (weight_fix(value_of<Bf16>(key_dropped) - vmax) != 0 || weight_fix(-256.0f - xmax) != 0)) return false;
    // a cut that shares its scaled value with entries that are not binned (a temperature that folds values together)
    auto shared_value = [&](uint32_t key, int q) {
        return (dropped && key <= key_dropped) || (n_mid > 0 && (q < HIST_SIDE ? key <= key_tiny : key >= key_tiny_neg));
    };
    if (f.use_k && shared_value(kstar, int(h.kpos))) return false;
    auto weight_of = [&](uint32_t key) { return weight_fix(key == kmax ? 0.0f : value_of<Bf16>(key) - vmax); };

    // ---- masses ----------------------------------------------------------------------------
    uint64_t mid = 0;
    for (int i = tid; i < int(n_tiny); i += S_THREADS) mid += weight_of(key_of_raw(h.tiny[i]));
    if (tid == 0 && n_zero) mid += n_zero * weight_of(key_of_raw(0));
    uint64_t mid_mass = 0;
    if (n_mid) block_excl_scan<uint64_t>(mid, h.wave_u64, &mid_mass);
    uint64_t m[HIST_PER], sum = 0, sum_raw = 0;
#pragma unroll
    for (int j = 0; j < HIST_PER; ++j) {
        const int q = tid * HIST_PER + j;
        m[j] = 0;
        sk[j] = 0;
        if (c[j] == 0) continue;
        if (q == HIST_SIDE) {
            m[j] = !f.use_k || int(h.kpos) > HIST_SIDE ? mid_mass : 0ull;
        } else {
            const uint32_t raw = raw_of_bin(bin_of_pos(q));
            sk[j] = key_of_raw(raw);
            const uint64_t w = weight_of(sk[j]) * c[j];
            if (sk[j] >= kstar) m[j] = w;
            if (want_lse) sum_raw += f.has_t ? weight_fix(Bf16::widen(uint16_t(raw)) - xmax) * c[j] : w;
        }
        sum += m[j];
    }
    uint64_t z_topk, z_raw = 0;
    uint64_t run = block_excl_scan<uint64_t>(sum, h.wave_u64, &z_topk);
    if (want_lse) {
        if (n_mid) {
            if (f.has_t) {
                for (int i = tid; i < int(n_tiny); i += S_THREADS) sum_raw += weight_fix(Bf16::widen(h.tiny[i]) - xmax);
                if (tid == 0 && n_zero) sum_raw += n_zero * weight_fix(-xmax);
            } else {
                sum_raw += mid;
            }
        }
        block_excl_scan<uint64_t>(sum_raw, h.wave_u64, &z_raw);
        // ln(z_raw 2^-40) + max: the masses round the row's exponentials down to 2^-40 of the largest, 1.2e-7 of the sum at most
        lse = double(xmax) + log(double(z_raw)) - FIX_BITS * 0.693147180559945309417232;
    }
    cut.kmax = kmax;
    cut.kstar = cut.kcut = kstar;
    cut.r_cut = 0xffffffffu;
    cut.z = z_topk;
    raw_cut = 0;
    if (!f.use_k && !f.use_p) return true;
    // ---- top-p -----------------------------------------------------------------------------
    if (f.use_p) {
        const uint64_t theta = floor_scale(f.top_p, z_topk);
        int best = -1;
        uint64_t upto = run;
#pragma unroll
        for (int j = 0; j < HIST_PER; ++j) {
            const int q = tid * HIST_PER + j;
            const bool in = c[j] > 0 && (q == HIST_SIDE ? (!f.use_k || int(h.kpos) > HIST_SIDE) : sk[j] >= kstar);
            if (in && upto <= theta) best = q;
            upto += m[j];
        }
        if (best >= 0) atomicMax(&h.best, uint32_t(best));
        __syncthreads();
        best = int(h.best);
        if (best == HIST_SIDE) return false;
        const uint32_t kcut = key_of_raw(raw_of_bin(bin_of_pos(best)));
        if (shared_value(kcut, best)) return false;
        upto = run;
#pragma unroll
        for (int j = 0; j < HIST_PER; ++j) {
            if (c[j] > 0 && sk[j] == kcut) {
                atomicAdd(&h.n_cut, c[j]);
                atomicMin(&h.before, (unsigned long long)upto);
            }
            upto += m[j];
        }
        __syncthreads();
        const uint32_t n_cut = h.n_cut;
        const uint64_t before = h.before, w_cut = weight_of(kcut);
        uint64_t r = n_cut;
        if (w_cut > 0) {
            const uint64_t fit = (theta - before) / w_cut + 1;  // entries t with before + t * w <= theta
            r = fit < r ? fit : r;
        }
        cut.kcut = kcut;
        cut.r_cut = r == n_cut ? 0xffffffffu : uint32_t(r);
        cut.z = before + r * w_cut;
    }
#pragma unroll
    for (int j = 0; j < HIST_PER; ++j)
        if (c[j] > 0 && sk[j] >= cut.kcut) atomicMax(&h.last, uint32_t(tid * HIST_PER + j));
    __syncthreads();
    raw_cut = masked_key<Bf16>(Bf16::widen(uint16_t(raw_of_bin(bin_of_pos(int(h.last))))));
    return true;
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

template <typename T>
__global__ __launch_bounds__(S_THREADS) __attribute__((amdgpu_waves_per_eu(4))) void verify_rows(VerifyParams p) {
    __shared__ VerifyShared lds;
    const int tid = threadIdx.x;
    const int64_t n_target = int64_t(p.batch) * (p.k + 1);
    const int64_t r = blockIdx.x;
    const bool is_target = r < n_target;
    const int per = is_target ? p.k + 1 : p.k;
    const int64_t q = is_target ? r : r - n_target;
    const int b = int(q / per), j = int(q % per);
    const int len = draft_len(p, b);
    if (j > len || (!is_target && j == len)) return;  // the whole workgroup: nobody reads this row's summary
    const typename T::raw_t *rp = is_target ? target_row<T>(p, b, j) : draft_row<T>(p, b, j);
    const bool vec = (is_target ? p.vec_target : p.vec_draft) != 0;
    const Filter f = filter_of(p, b);
    const bool want_lse = is_target && p.out_policy != nullptr;
    RowCut cut;
    uint32_t raw_cut = 0;
    double lse = 0.0;
    bool done = false;
    if constexpr (T::kDtype == KA_DTYPE_BF16) done = hist_cut(lds.hist, rp, p.vocab, f, want_lse, cut, raw_cut, lse);
    if (!done) {
        __syncthreads();
        cut = radix_cut<T>(lds.sh, rp, p.vocab, vec, f.temp, f.has_t, f.use_k, f.top_k, f.use_p, f.top_p, true);
        if (f.use_k || f.use_p) raw_cut = raw_key_of_cut<T>(cut.kcut, f.temp, f.has_t);
        if (want_lse) {
            row_lse_to_block<T>(rp, p.vocab, vec, lds.lse);
            __syncthreads();
            if (tid == 0) lse = lds.lse.value();
        }
    }

    // mass of the drafted token; where it sits in a tie group that survives in part, its rank in the group decides
    const int64_t d = j < len ? p.draft_ids[int64_t(b) * p.k + j] : -1;
    const bool in_vocab = d >= 0 && d < p.vocab;
    const uint32_t key = in_vocab ? elem_key<T>(rp[d], f.temp, f.has_t) : 0u;
    bool kept = in_vocab && (key > cut.kcut || (key == cut.kcut && key >= cut.kstar));
    if (kept && key == cut.kcut && cut.r_cut != 0xffffffffu) {  // the same for the whole block
        __syncthreads();
        if (tid == 0) lds.ties_before = 0;
        __syncthreads();
        uint32_t mine = 0;
        for_each_key<T>(rp, int(d), vec, f.temp, f.has_t, [&](int, uint32_t k) { mine += k == cut.kcut ? 1u : 0u; });
        if (mine) atomicAdd(&lds.ties_before, mine);
        __syncthreads();
        kept = lds.ties_before < cut.r_cut;
    }
    if (tid == 0) {
        RowSummary s;
        s.z = cut.z;
        s.w_draft = kept ? weight_fix(key == cut.kmax ? 0.0f : value_of<T>(key) - value_of<T>(cut.kmax)) : 0ull;
        s.lse = lse;
        s.kmax = cut.kmax;
        s.kcut = cut.kcut;
        s.r_cut = cut.r_cut;
        s.raw_cut = raw_cut;
        p.rows[r] = s;
    }
}

// ---------------------------------------------------------------------------
// verify_ties: grid (B, 2).  Where a row's cut falls inside a tie group, the index below which the group's entries survive:
// the ties of every chunk of 512 vectors are counted, and the chunk that holds the last survivor is read once more in order.
// ---------------------------------------------------------------------------
constexpr int MAX_CHUNKS = (1 << 22) / (4 * S_THREADS);
template <typename T>
__global__ __launch_bounds__(S_THREADS) void verify_ties(VerifyParams p) {
    __shared__ uint32_t ties[MAX_CHUNKS];
    __shared__ uint32_t wave_buf[S_WAVES];
    __shared__ uint32_t s_chunk, s_before;
    constexpr int EPV = T::kPerVec;
    const int b = blockIdx.x, tid = threadIdx.x;
    const bool is_target = blockIdx.y == 0;
    const int len = draft_len(p, b);
    const int n = accepted_prefix(p, b, len);
    if (!is_target && (n == len || p.draft == nullptr)) return;
    const int64_t row = is_target ? int64_t(b) * (p.k + 1) + n : int64_t(p.batch) * (p.k + 1) + int64_t(b) * p.k + n;
    const uint32_t r_cut = p.rows[row].r_cut, kcut = p.rows[row].kcut;
    int32_t *const limit = p.tie_limit + 2 * b + (is_target ? 0 : 1);
    if (r_cut == 0xffffffffu) {
        if (tid == 0) *limit = 0x7fffffff;
        return;
    }
    const Filter f = filter_of(p, b);
    const typename T::raw_t *rp = is_target ? target_row<T>(p, b, n) : draft_row<T>(p, b, n);
    const bool vec = (is_target ? p.vec_target : p.vec_draft) != 0;
    const float low = cut_value<T>(p.rows[row].raw_cut);
    auto ties_of = [&](const typename T::raw_t (&e)[EPV], int base) {
        uint32_t c = 0;
#pragma unroll
        for (int j = 0; j < EPV; ++j)
            if (!(T::widen(e[j]) < low) && base + j < p.vocab && elem_key<T>(e[j], f.temp, f.has_t) == kcut) ++c;
        return c;
    };
    const int chunks = (p.vocab + EPV * S_THREADS - 1) / (EPV * S_THREADS);
    for (int i = tid; i < chunks; i += S_THREADS) ties[i] = 0;
    __syncthreads();
    constexpr int U = 8;  // vectors in flight per lane
    for (int c0 = 0; c0 < chunks; c0 += U) {
        typename T::raw_t e[U][EPV];
#pragma unroll
        for (int u = 0; u < U; ++u) load_entries<T>(rp, vec, p.vocab, ((c0 + u) * S_THREADS + tid) * int64_t(EPV), e[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t base = ((c0 + u) * S_THREADS + tid) * int64_t(EPV);
            if (base >= p.vocab) continue;
            const uint32_t c = ties_of(e[u], int(base));
            if (c) atomicAdd(&ties[c0 + u], c);
        }
    }
    __syncthreads();
    // chunks in order: thread t takes a run of them
    const int per = (chunks + S_THREADS - 1) / S_THREADS;
    uint32_t mine = 0, total;
    for (int i = 0; i < per; ++i) mine += tid * per + i < chunks ? ties[tid * per + i] : 0u;
    const uint32_t before = block_excl_scan<uint32_t>(mine, wave_buf, &total);
    if (before < r_cut && r_cut <= before + mine) {
        uint32_t at = before;
        for (int i = 0; i < per; ++i) {
            const uint32_t c = ties[tid * per + i];
            if (r_cut <= at + c) { s_chunk = uint32_t(tid * per + i); s_before = at; break; }
            at += c;
        }
    }
    __syncthreads();
    const int64_t base = (int64_t(s_chunk) * S_THREADS + tid) * EPV;
    typename T::raw_t e[EPV];
    load_entries<T>(rp, vec, p.vocab, base, e);
    const uint32_t c = base < p.vocab ? ties_of(e, int(base)) : 0u;
    const uint32_t rank = s_before + block_excl_scan<uint32_t>(c, wave_buf, &total);
    if (rank < r_cut && r_cut <= rank + c) {
        uint32_t at = rank;
        int32_t found = 0;
#pragma unroll
        for (int j = 0; j < EPV; ++j)
            if (base + j < p.vocab && elem_key<T>(e[j], f.temp, f.has_t) == kcut && ++at == r_cut) found = int32_t(base) + j + 1;
        *limit = found;
    }
}

// ---------------------------------------------------------------------------
// Residual masses of the stopping position
// ---------------------------------------------------------------------------
// A row's distribution as the last two kernels evaluate it, entry by entry.
struct RowDist {
    uint32_t kmax, kcut;
    int limit;
    float vmax;
    template <typename T> __device__ __forceinline__ uint64_t mass(uint32_t key, int i) const {
        if (key < kcut || (key == kcut && i >= limit)) return 0ull;
        return weight_fix(key == kmax ? 0.0f : value_of<T>(key) - vmax);
    }
};

// Residual mass of entry i: max(W^p mul_p - W^q mul_q, 0), 0 for a looked-up draft that was rejected.
template <typename T> struct Residual {
    const typename T::raw_t *rp, *rq;  // rq null: nothing is subtracted
    bool vec_p, vec_q;
    RowDist p, q;
    float low_p, low_q;  // unscaled values below these have no mass
    uint64_t mul_p, mul_q;
    int64_t skip;  // the rejected look-up draft, or -1
    Filter f;
    int vocab;

    __device__ __forceinline__ void setup(const VerifyParams &v, int b, int n, int len) {
        const RowSummary &t = v.rows[int64_t(b) * (v.k + 1) + n];
        f = filter_of(v, b);
        vocab = v.vocab;
        rp = target_row<T>(v, b, n);
        vec_p = v.vec_target != 0;
        p = RowDist{t.kmax, t.kcut, v.may_cut_ties ? v.tie_limit[2 * b] : 0x7fffffff, value_of<T>(t.kmax)};
        mul_p = 1;
        mul_q = 0;
        rq = nullptr;
        vec_q = false;
        skip = -1;
        q = p;
        low_p = low_q = cut_value<T>(t.raw_cut);
        if (n < len) {
            if (v.draft != nullptr) {
                const RowSummary &d = v.rows[int64_t(v.batch) * (v.k + 1) + int64_t(b) * v.k + n];
                rq = draft_row<T>(v, b, n);
                vec_q = v.vec_draft != 0;
                q = RowDist{d.kmax, d.kcut, v.may_cut_ties ? v.tie_limit[2 * b + 1] : 0x7fffffff, value_of<T>(d.kmax)};
                low_q = cut_value<T>(d.raw_cut);
                mul_p = d.z;
                mul_q = t.z;
            } else {
                skip = v.draft_ids[int64_t(b) * v.k + n];
            }
        }
    }
    __device__ __forceinline__ u128 entry(typename T::raw_t x, typename T::raw_t y, int i) const {
        if (T::widen(x) < low_p || i >= vocab || int64_t(i) == skip) return 0;
        const uint64_t wp = p.template mass<T>(elem_key<T>(x, f.temp, f.has_t), i);
        if (wp == 0) return 0;
        if (rq == nullptr) return wp;
        const u128 have = u128(wp) * mul_p;
        if (T::widen(y) < low_q) return have;
        const u128 take = u128(q.template mass<T>(elem_key<T>(y, f.temp, f.has_t), i)) * mul_q;
        return have > take ? have - take : u128(0);
    }
    // residual masses of the vector that starts at `base` (0 behind the row)
    __device__ __forceinline__ void vector(int64_t base, u128 (&m)[T::kPerVec]) const {
        constexpr int EPV = T::kPerVec;
        typename T::raw_t x[EPV], y[EPV];
        load_entries<T>(rp, vec_p, vocab, base, x);
        if (rq != nullptr) load_entries<T>(rq, vec_q, vocab, base, y);
#pragma unroll
        for (int j = 0; j < EPV; ++j) m[j] = base + j < vocab ? entry(x[j], rq != nullptr ? y[j] : typename T::raw_t(0), int(base) + j) : u128(0);
    }
};

// The entry of a vector of masses, `before` of mass in front of it, that holds tau.
template <int EPV> __device__ __forceinline__ int entry_at(const u128 (&m)[EPV], u128 before, u128 tau) {
    int hit = -1;
#pragma unroll
    for (int j = 0; j < EPV; ++j) {
        before += m[j];
        if (hit < 0 && tau < before) hit = j;
    }
    return hit;
}
template <int EPV> __device__ __forceinline__ u128 total_of(const u128 (&m)[EPV]) {
    u128 sum = 0;
#pragma unroll
    for (int j = 0; j < EPV; ++j) sum += m[j];
    return sum;
}

__device__ __forceinline__ u128 shfl_up_u128(u128 v, int off) {
    const uint64_t lo = __shfl_up((unsigned long long)uint64_t(v), off, kWave);
    const uint64_t hi = __shfl_up((unsigned long long)uint64_t(v >> 64), off, kWave);
    return (u128(hi) << 64) | lo;
}
__device__ __forceinline__ u128 wave_incl_scan_u128(u128 v) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const u128 o = shfl_up_u128(v, off);
        if (lane >= off) v += o;
    }
    return v;
}
// Exclusive prefix sum over the block in thread order; `*total` = sum over the block.  Every thread calls it.
template <int WAVES> __device__ __forceinline__ u128 block_excl_scan_u128(u128 v, u128 *wave_buf, u128 *total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const u128 inc = wave_incl_scan_u128(v);
    __syncthreads();  // wave_buf may still be read from a previous call
    if (lane == kWave - 1) wave_buf[wave] = inc;
    __syncthreads();
    u128 base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const u128 x = wave_buf[w];
        if (w < wave) base += x;
        sum += x;
    }
    *total = sum;
    return base + inc - v;
}

// grid (groups of shares, B): a wavefront per share
template <typename T>
__global__ __launch_bounds__(SHARE_THREADS) void verify_shares(VerifyParams p) {
    const int b = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    const int share = int(blockIdx.x) * (SHARE_THREADS / kWave) + int(threadIdx.x) / kWave;
    const int len = draft_len(p, b);
    const int n = accepted_prefix(p, b, len);
    if (share >= p.n_shares) return;
    Residual<T> res;
    res.setup(p, b, n, len);
    u128 sum = 0;
#pragma unroll 1
    for (int s = 0; s < SHARE_VECS / kWave; ++s) {
        const int64_t base = (int64_t(share) * SHARE_VECS + s * kWave + lane) * T::kPerVec;
        u128 m[T::kPerVec];
        res.vector(base, m);
        sum += total_of(m);
    }
    sum = wave_incl_scan_u128(sum);
    if (lane == kWave - 1) p.shares[int64_t(b) * p.n_shares + share] = sum;
}

// grid B; a thread per vector of the share that holds the draw
template <typename T>
__global__ __launch_bounds__(SHARE_VECS) void verify_draw(VerifyParams p) {
    constexpr int WAVES = SHARE_VECS / kWave;
    __shared__ u128 wave_buf[WAVES];
    __shared__ u128 s_before;
    __shared__ int s_share, s_hit;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int len = draft_len(p, b);
    const int n = accepted_prefix(p, b, len);
    if (tid == 0) { s_share = -1; s_hit = -1; }
    const float u = clean_uniform(p.uniforms[int64_t(b) * (p.k + 1) + p.k]);
    // the share that holds floor(u * R): thread t takes a run of shares
    u128 mine = 0, r;
    const int per = (p.n_shares + SHARE_VECS - 1) / SHARE_VECS;
    const u128 *const shares = p.shares + int64_t(b) * p.n_shares;
    for (int i = 0; i < per; ++i)
        if (tid * per + i < p.n_shares) mine += shares[tid * per + i];
    const u128 excl = block_excl_scan_u128<WAVES>(mine, wave_buf, &r);
    u128 tau = floor_scale_wide(u, r);
    if (excl <= tau && tau < excl + mine) {
        u128 at = excl;
        for (int i = 0; i < per; ++i) {
            const u128 m = shares[tid * per + i];
            if (tau < at + m) { s_share = tid * per + i; s_before = at; break; }
            at += m;
        }
    }
    Residual<T> res;
    res.setup(p, b, n, len);
    __syncthreads();
    int share = s_share, last = share;
    u128 at = share >= 0 ? s_before : u128(0);
    if (r == 0) {  // no residual (see the head of the file): drawn from P, share after share
        res.rq = nullptr;
        res.skip = -1;
        tau = floor_scale_wide(u, p.rows[int64_t(b) * (p.k + 1) + n].z);
        share = 0;
        last = p.n_shares - 1;
    }
    for (; share >= 0 && share <= last; ++share) {  // block-uniform, one turn unless r is 0
        const int64_t base = (int64_t(share) * SHARE_VECS + tid) * T::kPerVec;
        u128 m[T::kPerVec], total;
        res.vector(base, m);
        const u128 sum = total_of(m);
        const u128 before = at + block_excl_scan_u128<WAVES>(sum, wave_buf, &total);
        if (before <= tau && tau < before + sum) s_hit = int(base) + entry_at(m, before, tau);
        at += total;
        if (tau < at) break;
    }
    __syncthreads();
    // outputs: lane j writes position j
    for (int j = tid; j <= p.k; j += SHARE_VECS) {
        const int64_t at = int64_t(b) * (p.k + 1) + j;
        const int64_t id = j < n ? p.draft_ids[int64_t(b) * p.k + j] : (j == n ? int64_t(s_hit) : int64_t(-1));
        p.out_ids[at] = id;
        if (p.out_policy != nullptr) {
            float lp = 0.0f;
            if (j <= n) lp = id >= 0 ? float(double(T::widen(target_row<T>(p, b, j)[id])) - p.rows[at].lse) : __builtin_nanf("");
            p.out_policy[at] = lp;
        }
    }
    if (tid == 0) p.out_accepted[b] = n;
}

template <typename T> int launch_verify(const VerifyParams &p, hipStream_t stream) {
    const int64_t rows = int64_t(p.batch) * (p.k + 1) + (p.draft != nullptr ? int64_t(p.batch) * p.k : 0);
    hipLaunchKernelGGL((verify_rows<T>), dim3(unsigned(rows)), dim3(S_THREADS), 0, stream, p);
    int rc = check_hip(hipGetLastError(), "verify launch (rows)");
    if (rc != KA_OK) return rc;
    if (p.may_cut_ties) {
        hipLaunchKernelGGL((verify_ties<T>), dim3(unsigned(p.batch), 2), dim3(S_THREADS), 0, stream, p);
        rc = check_hip(hipGetLastError(), "verify launch (ties)");
        if (rc != KA_OK) return rc;
    }
    hipLaunchKernelGGL((verify_shares<T>), dim3(unsigned((p.n_shares * kWave + SHARE_THREADS - 1) / SHARE_THREADS), unsigned(p.batch)), dim3(SHARE_THREADS), 0, stream, p);
    rc = check_hip(hipGetLastError(), "verify launch (shares)");
    if (rc != KA_OK) return rc;
    hipLaunchKernelGGL((verify_draw<T>), dim3(unsigned(p.batch)), dim3(SHARE_VECS), 0, stream, p);
    return check_hip(hipGetLastError(), "verify launch (draw)");
}

inline size_t align_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

struct VerifyLayout {
    int64_t n_shares;
    size_t rows, ties, shares, total;
};
inline VerifyLayout verify_layout(int dtype, int64_t batch, int64_t k, int64_t vocab) {
    VerifyLayout l;
    const int64_t epv = dtype == KA_DTYPE_F32 ? 4 : 8;
    l.n_shares = (vocab + SHARE_VECS * epv - 1) / (SHARE_VECS * epv);
    l.rows = 0;
    l.ties = align_up(size_t(batch) * size_t(2 * k + 1) * sizeof(RowSummary), 256);
    l.shares = l.ties + align_up(size_t(batch) * 8, 256);
    l.total = l.shares + size_t(batch) * size_t(l.n_shares) * sizeof(u128);
    return l;
}

}  // namespace
}  // namespace ka

KA_EXPORT size_t ka_verify_workspace_bytes(int dtype, int64_t batch, int64_t max_draft, int64_t vocab) {
    if (batch <= 0 || max_draft < 0 || max_draft > ka::VERIFY_MAX_DRAFT || vocab < 1 || vocab >= (int64_t(1) << 22)) return 0;
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
    if (vocab >= (int64_t(1) << 22))
        return fail(KA_ERR_UNSUPPORTED, "verify: vocab %lld >= 2^22 (integer masses would overflow)", (long long)vocab);
    if (batch > 65535) return fail(KA_ERR_UNSUPPORTED, "verify: batch %lld > 65535", (long long)batch);
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
    p.tie_limit = reinterpret_cast<int32_t *>(ws + l.ties);
    p.shares = reinterpret_cast<u128 *>(ws + l.shares);
    p.n_shares = int32_t(l.n_shares);
    auto aligned = [&](const void *base, int64_t batch_stride, int64_t pos_stride, int64_t positions) {
        return reinterpret_cast<uintptr_t>(base) % 16 == 0 && (batch == 1 || (batch_stride * esize) % 16 == 0) &&
               (positions <= 1 || (pos_stride * esize) % 16 == 0);
    };
    p.vec_target = aligned(target_logits, target_batch_stride, target_pos_stride, max_draft + 1) ? 1 : 0;
    p.vec_draft = p.draft != nullptr && aligned(draft_logits, draft_batch_stride, draft_pos_stride, max_draft) ? 1 : 0;
    p.may_cut_ties = (top_p_rows != nullptr || top_p < 1.0f) ? 1 : 0;
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    if (dtype == KA_DTYPE_BF16) return launch_verify<Bf16>(p, stream);
    if (dtype == KA_DTYPE_F16) return launch_verify<F16>(p, stream);
    return launch_verify<F32>(p, stream);
}
