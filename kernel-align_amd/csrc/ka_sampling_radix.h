// The radix path of the sampling kernels up to the draw: which entries of a row survive top-k and top-p, and their mass.
#ifndef KA_SAMPLING_RADIX_H
#define KA_SAMPLING_RADIX_H

#include "ka_sampling_common.h"

namespace ka {
namespace {

// The distribution of a row after temperature, top-k and top-p.  Survivors: key > kcut, and of the entries equal to kcut
// the first r_cut in index order (0xffffffff: all of them).
struct RowCut {
    uint32_t kmax;   // largest key
    uint32_t kstar;  // top-k keeps key >= kstar
    uint32_t kcut, r_cut;
    uint64_t z;      // integer mass of the survivors (not filled without need_z and top-p)
};

// Every thread of the block calls this with the same arguments; it contains barriers.  Any row, any parameters: 2 + LEVELS
// (top-k) + LEVELS (top-p) passes over the row.
template <typename T>
__device__ __forceinline__ RowCut radix_cut(Shared &sh, const typename T::raw_t *rp, int vocab, bool vec, float temp,
                                            bool has_t, bool use_k, int top_k, bool use_p, float top_p, bool need_z) {
    constexpr int LEVELS = Round<T>::kLevels;
    const int tid = threadIdx.x;
    // ---- pass 0: row maximum and the level-0 count histogram --------------------------
    clear_hist(sh);
    __syncthreads();
    uint32_t kmax = 0;
    for_each_key<T>(rp, vocab, vec, temp, has_t, [&](int, uint32_t key) {
        kmax = key > kmax ? key : kmax;
        if (use_k) atomicAdd(&sh.h.cnt[key >> 21], 1u);
    });
    kmax = block_max_u32(kmax, sh);  // barriers inside also publish the histogram
    const float vmax = value_of<T>(kmax);

    // ---- top-k: MSB-first descent to the k-th largest key --------------------------------
    uint32_t kstar = 0;      // keep key >= kstar
    uint32_t n_eq_kstar = 0; // entries equal to kstar (only meaningful with use_k)
    if (use_k) {
        uint32_t rank = uint32_t(top_k);  // 1-based rank inside the current prefix
        uint32_t prefix = 0;
        for (int level = 0; level < LEVELS; ++level) {
            const int shift = level_shift<T>(level), bits = level_bits<T>(level);
            const uint32_t nb = 1u << bits;
            if (level > 0) {
                clear_hist(sh);
                __syncthreads();
                const int pshift = level_shift<T>(level - 1);
                for_each_key<T>(rp, vocab, vec, temp, has_t, [&](int, uint32_t key) {
                    if ((key >> pshift) == prefix) atomicAdd(&sh.h.cnt[(key >> shift) & (nb - 1)], 1u);
                });
                __syncthreads();
            }
            uint32_t above;
            const uint32_t digit = select_count_bin(sh, nb, rank, &above, &n_eq_kstar);
            prefix = (prefix << bits) | digit;
            rank -= above;
        }
        kstar = prefix << level_shift<T>(LEVELS - 1);
    }

    // ---- masses of the survivors of top-k: total, and level-0 histogram for top-p ---------
    uint64_t z_topk = 0;
    if (need_z || use_p) {
        clear_hist(sh);
        __syncthreads();
        uint64_t zpart = 0;
        for_each_key<T>(rp, vocab, vec, temp, has_t, [&](int, uint32_t key) {
            if (key >= kstar) {
                const float y = value_of<T>(key);
                const uint64_t w = weight_fix(key == kmax ? 0.0f : y - vmax);
                zpart += w;
                if (use_p) {
                    atomicAdd(reinterpret_cast<unsigned long long *>(&sh.h.mass[key >> 21]), (unsigned long long)w);
                    atomicAdd(&sh.h.cnt[key >> 21], 1u);
                }
            }
        });
        block_excl_scan<uint64_t>(zpart, sh.wave_u64, &z_topk);
        __syncthreads();
    }

    // ---- top-p: descent to the lowest key whose first entry is still kept ------------------
    uint32_t kcut = kstar;            // survivors: key > kcut, or key == kcut with tie rank < r_cut
    uint32_t r_cut = 0xffffffffu;
    uint64_t z_kept = z_topk;
    if (use_p) {
        const uint64_t theta = floor_scale(top_p, z_topk);
        uint64_t before = 0;          // mass of the keys above the current prefix
        uint32_t prefix = 0;
        uint32_t n_cut = 0;
        uint64_t m_cut = 0;
        for (int level = 0; level < LEVELS; ++level) {
            const int shift = level_shift<T>(level), bits = level_bits<T>(level);
            const uint32_t nb = 1u << bits;
            if (level > 0) {
                clear_hist(sh);
                __syncthreads();
                const int pshift = level_shift<T>(level - 1);
                for_each_key<T>(rp, vocab, vec, temp, has_t, [&](int, uint32_t key) {
                    if (key >= kstar && (key >> pshift) == prefix) {
                        const float y = value_of<T>(key);
                        const uint64_t w = weight_fix(key == kmax ? 0.0f : y - vmax);
                        const uint32_t d = (key >> shift) & (nb - 1);
                        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.h.mass[d]), (unsigned long long)w);
                        atomicAdd(&sh.h.cnt[d], 1u);
                    }
                });
                __syncthreads();
            }
            // thread t owns the bins BINS_PER_THREAD * t + j counted from the top
            uint64_t m[BINS_PER_THREAD], mine = 0;
            uint32_t c[BINS_PER_THREAD];
#pragma unroll
            for (int j = 0; j < BINS_PER_THREAD; ++j) {
                const int rb = BINS_PER_THREAD * tid + j;
                m[j] = rb < int(nb) ? sh.h.mass[nb - 1 - rb] : 0ull;
                c[j] = rb < int(nb) ? sh.h.cnt[nb - 1 - rb] : 0u;
                mine += m[j];
            }
            uint64_t total;
            const uint64_t excl = block_excl_scan<uint64_t>(mine, sh.wave_u64, &total);
            if (tid == 0) sh.best_rb = -1;
            __syncthreads();
            {   // the lowest of the thread's occupied bins whose first entry is still kept
                int mine_rb = -1;
                uint64_t run = excl;
#pragma unroll
                for (int j = 0; j < BINS_PER_THREAD; ++j) {
                    if (c[j] > 0 && before + run <= theta) mine_rb = BINS_PER_THREAD * tid + j;
                    run += m[j];
                }
                if (mine_rb >= 0) atomicMax(&sh.best_rb, mine_rb);
            }
            __syncthreads();
            const int best = sh.best_rb;
            {
                uint64_t run = excl;
#pragma unroll
                for (int j = 0; j < BINS_PER_THREAD; ++j) {
                    if (best == BINS_PER_THREAD * tid + j) { sh.sel_mass_above = run; sh.sel_mass = m[j]; sh.sel_count = c[j]; }
                    run += m[j];
                }
            }
            __syncthreads();
            prefix = (prefix << bits) | uint32_t(nb - 1 - best);
            before += sh.sel_mass_above;
            n_cut = sh.sel_count;
            m_cut = sh.sel_mass;
            __syncthreads();
        }
        kcut = prefix << level_shift<T>(LEVELS - 1);
        const uint64_t w_cut = n_cut ? m_cut / n_cut : 0;   // every entry of the tie group has this mass
        uint64_t r = n_cut;
        if (w_cut > 0) {
            const uint64_t fit = (theta - before) / w_cut + 1;  // entries t with before + t*w <= theta
            r = fit < r ? fit : r;
        }
        r_cut = uint32_t(r);
        z_kept = before + r * w_cut;
        if (r == n_cut) r_cut = 0xffffffffu;  // whole tie group survives: no rank bookkeeping needed
    }
    return RowCut{kmax, kstar, kcut, r_cut, z_kept};
}

}  // namespace
}  // namespace ka

#endif  // KA_SAMPLING_RADIX_H
