// Low-rank adapters of many requests beside a shared projection, forward and backward.
//
//   forward    u_n = s_a x_n A_a^T           y_n = base_n + u_n B_a^T             a = adapter_ids[n], none: y_n = base_n
//   backward   du_n = s_a dy_n B_a           dx_n = dx_base_n + du_n A_a
//              dA_a = sum_n du_n^T x_n       dB_a = sum_n dy_n^T u_n              over the tokens n of adapter a, in order
//
// x [N, H], base / y / dy [N, O], A [S, R, H], B [S, O, R], R <= 128.  The tokens are sorted by adapter on the device (a stable
// counting sort, lora_plan) and worked on in tiles of one adapter each, so that every product is a small dense one on the
// matrix cores (v_mfma_f32_16x16x32).  All of it is bound by memory: per token 2 H bytes in and 4 O bytes through for
// 2 R (H + O) flop, 16 flop per byte at R = 16, against about 300 that the matrix cores could do.
//
// Numbers.  Products of two 16-bit matrices (x A^T, dy B) run in their own type with fp32 accumulation.  u and du are fp32 and
// stay so: next to a 16-bit matrix they are split into bf16 parts, high + low (17 bits: for results that are rounded
// to 16 bits) or high + middle + low (24 bits: for the fp32 gradients), and an fp16 matrix into the two bf16 that hold it exactly (11
// bits).  bf16 has fp32's range, so the bits are each entry's own: fp16 parts of u would share one scale per token, and a small
// u_r beside a large one would lose its bits however large its column of B.
// Every sum runs in a fixed order: no atomics on floating-point values.
// Infinities come out as in the definition.  The low parts of a number are 0 or of either sign, so that a product of parts with an
// infinity is no number; where such a sum is not finite it is formed again from the leading parts alone, which are 0, infinite and of
// a sign as the numbers are, without the places that a lane without work reads (leading_kind).  To see that nothing has to be costs
// one instruction a sum: backward of 2048 x 4096, us a call without and with it, rank 16 57.1 / 57.7, rank 128 164 / 170.
#include <type_traits>

#include "ka_common.h"

namespace ka {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int MAX_RANK = KA_LORA_MAX_RANK;
constexpr int MAX_ADAPTERS = KA_LORA_MAX_ADAPTERS;
constexpr int THREADS = 256;
constexpr int WAVES = THREADS / kWave;
constexpr int FWD_TILE = 32;    // tokens per tile of the forward: two groups of sixteen
constexpr int FWD_SUBS = FWD_TILE / 16;
static_assert(KA_LORA_MAX_TOKENS / FWD_TILE + MAX_ADAPTERS + 1 <= 65535, "the tiles are the second dimension of a grid");
constexpr int BWD_TILE_MAX = 1024;  // ... of the backward at most (a multiple of 32)

struct LoraTile {
    int32_t adapter;       // -1: tokens without one
    int32_t start, count;  // in `order`
    int32_t slot;          // backward: -1 writes the adapter's gradient, others this partial one
};
struct TileList {
    int32_t *count;        // [1]
    LoraTile *tiles;
    int32_t *per_adapter;  // [2 S]: tiles of the adapter, its first partial slot
    int32_t tokens;        // per tile
};
struct LoraPlan {          // device pointers into the workspace
    int32_t *order;        // [N] tokens sorted by adapter, those without one last
    TileList list[2];      // of the forward, or of the backward's two passes
};

// ---------------------------------------------------------------------------
// lora_plan: one workgroup sorts the tokens.  Every wavefront takes a contiguous share of them: counts, a prefix over
// (adapter, wavefront), then the ranks inside a step of 64 tokens from ballots.  The ids of eight steps are requested together.
// One workgroup, since a sort over several would need launches of its own: bound by its chain of waits, 6 us for 777 tokens, 8 for
// 2048, 15 for 5003.
// ---------------------------------------------------------------------------
template <int PLAN_THREADS> struct PlanShared {
    int32_t at[PLAN_THREADS / kWave][MAX_ADAPTERS + 1];  // counts, then the next position of the wavefront's tokens
    int32_t wave_sum[PLAN_THREADS / kWave][5];
};
template <int PLAN_THREADS>
__device__ __forceinline__ void make_plan(PlanShared<PLAN_THREADS> &sh, const int64_t *__restrict__ ids, int n, int s, int lists, const LoraPlan &plan) {
    constexpr int PLAN_WAVES = PLAN_THREADS / kWave;
    auto &at = sh.at;
    auto &wave_sum = sh.wave_sum;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    constexpr int U = 8;
    const int steps = (n + kWave - 1) / kWave, per = (steps + PLAN_WAVES - 1) / PLAN_WAVES;
    const int s0 = wave * per, s1 = s0 + per < steps ? s0 + per : steps;
    int a[U];  // adapters of eight steps of this wavefront; s: none, -1: behind the end
    auto load = [&](int st) {
        int64_t id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (st + u) * kWave + lane;
            id[u] = st + u < s1 && i < n ? ids[i] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (st + u) * kWave + lane;
            a[u] = st + u < s1 && i < n ? (id[u] >= 0 && id[u] < s ? int(id[u]) : s) : -1;
        }
    };
    load(s0);
    for (int i = tid; i < PLAN_WAVES * (s + 1); i += PLAN_THREADS) at[i / (s + 1)][i % (s + 1)] = 0;
    __syncthreads();
    for (int st = s0; st < s1; st += U) {
        if (st != s0) load(st);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (a[u] >= 0) atomicAdd(&at[wave][a[u]], 1);
    }
    __syncthreads();
    // thread t owns the adapters t * own .. : tokens, and per list tiles and partial slots, before its first
    const int own = (s + 1 + PLAN_THREADS - 1) / PLAN_THREADS;
    int mine[5] = {0, 0, 0, 0, 0};
    for (int j = 0; j < own; ++j) {
        const int ad = tid * own + j;
        if (ad > s) break;
        int c = 0;
        for (int w = 0; w < PLAN_WAVES; ++w) c += at[w][ad];
        mine[0] += c;
        for (int l = 0; l < lists; ++l) {
            const int t = (c + plan.list[l].tokens - 1) / plan.list[l].tokens;
            mine[1 + 2 * l] += t;
            if (ad < s && t > 1) mine[2 + 2 * l] += t - 1;
        }
    }
    int before[5];
#pragma unroll
    for (int q = 0; q < 5; ++q) {
        int inc = mine[q];
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const int o = __shfl_up(inc, off, kWave);
            if (lane >= off) inc += o;
        }
        if (lane == kWave - 1) wave_sum[wave][q] = inc;
        before[q] = inc - mine[q];
    }
    __syncthreads();
    int total[2] = {0, 0};
    for (int w = 0; w < PLAN_WAVES; ++w) {
        if (w < wave) {
#pragma unroll
            for (int q = 0; q < 5; ++q) before[q] += wave_sum[w][q];
        }
        total[0] += wave_sum[w][1];
        total[1] += wave_sum[w][3];
    }
    for (int j = 0; j < own; ++j) {
        const int ad = tid * own + j;
        if (ad > s) break;
        int c = 0;
        for (int w = 0; w < PLAN_WAVES; ++w) {
            const int x = at[w][ad];
            at[w][ad] = before[0] + c;
            c += x;
        }
#pragma unroll
        for (int l = 0; l < 2; ++l) {
            if (l >= lists) break;
            const TileList &list = plan.list[l];
            const int t = (c + list.tokens - 1) / list.tokens;
            for (int k = 0; k < t; ++k) {
                LoraTile lt;
                lt.adapter = ad < s ? ad : -1;
                lt.start = before[0] + k * list.tokens;
                lt.count = c - k * list.tokens < list.tokens ? c - k * list.tokens : list.tokens;
                lt.slot = k == 0 ? -1 : before[2 + 2 * l] + k - 1;
                list.tiles[before[1 + 2 * l] + k] = lt;
            }
            if (ad < s) {
                list.per_adapter[2 * ad] = t;
                list.per_adapter[2 * ad + 1] = before[2 + 2 * l];
            }
            before[1 + 2 * l] += t;
            if (ad < s && t > 1) before[2 + 2 * l] += t - 1;
        }
        before[0] += c;
    }
    if (tid < lists) *plan.list[tid].count = total[tid];
    __syncthreads();
    for (int st = s0; st < s1; st += U) {
        if (per > U) load(st);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint64_t left = __ballot(a[u] >= 0);
            while (left != 0) {  // one turn per adapter that occurs in the step
                const int leader = __ffsll((long long)left) - 1;
                const int want = __builtin_amdgcn_readlane(a[u], leader);
                const uint64_t same = __ballot(a[u] == want);
                const int base = at[wave][want];
                if (a[u] == want) plan.order[base + __popcll(same & ((uint64_t(1) << lane) - 1))] = (st + u) * kWave + lane;
                // the wavefront's own counter: read by all lanes above, moved by one
                __builtin_amdgcn_wave_barrier();
                if (lane == leader) at[wave][want] = base + __popcll(same);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                left &= ~same;
            }
        }
    }
}
constexpr int PLAN_THREADS = 512;
__global__ __launch_bounds__(PLAN_THREADS) void lora_plan(const int64_t *__restrict__ ids, int n, int s, int lists, LoraPlan plan) {
    __shared__ PlanShared<PLAN_THREADS> sh;
    make_plan(sh, ids, n, s, lists, plan);
}

// ---------------------------------------------------------------------------
// Fragments.  v_mfma_f32_16x16x32: lane l holds eight values (one 16-byte register group) of row / column l % 16 at the
// contraction indices 8 (l / 16) .. + 7 of either operand; the result's lane l holds column l % 16, rows 4 (l / 16) .. + 3.
// ---------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ f32x4 mfma(const uint4 &a, const uint4 &b, const f32x4 &c) {
    if constexpr (T::kDtype == KA_DTYPE_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    bf16x2 v;
    v[0] = __bf16(lo);
    v[1] = __bf16(hi);
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// What rounding to bf16 left of a value; 0 behind an infinity or NaN, which the high part carries alone.
__device__ __forceinline__ float rest(float v, float part) { return fabsf(part) < __builtin_inff() ? v - part : 0.0f; }

// v = part[0] + part[1] (+ part[2]) in bf16: relative error 2^-17 with two parts, none (24 bits) with three
template <int PARTS> __device__ __forceinline__ void split(const float (&v)[8], uint4 (&part)[PARTS]) {
    uint32_t w[PARTS][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a = v[2 * j], b = v[2 * j + 1];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            w[p][j] = pack_bf16(a, b);
            a = rest(a, low_half(w[p][j]));
            b = rest(b, high_half(w[p][j]));
        }
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p) part[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}
__device__ __forceinline__ uint4 choose(bool first, const uint4 &a, const uint4 &b) {
    return make_uint4(first ? a.x : b.x, first ? a.y : b.y, first ? a.z : b.z, first ? a.w : b.w);
}
// A fragment of the data's type as bf16 parts: itself, or the two that hold an fp16 exactly.
template <typename T> struct Parts { static constexpr int kCount = T::kDtype == KA_DTYPE_BF16 ? 1 : 2; };
template <typename T> __device__ __forceinline__ void as_bf16(const uint4 &f, uint4 (&part)[Parts<T>::kCount]) {
    if constexpr (T::kDtype == KA_DTYPE_BF16) {
        part[0] = f;
    } else {
        // an fp16 has 11 bits: the 8 of its first half as fp32, and the 3 that are left, which fp32's subtraction gives exactly
        float v[8];
        F16::unpack(f, v);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = __float_as_uint(v[2 * j]), b = __float_as_uint(v[2 * j + 1]);
            hi[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            lo[j] = __builtin_amdgcn_perm(__float_as_uint(v[2 * j + 1] - high_half(b)), __float_as_uint(v[2 * j] - high_half(a)), 0x07060302u);
        }
        part[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        part[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// Whether a sum of some lane of the wavefront is not finite (the same in every lane).
__device__ __forceinline__ bool any_odd(const f32x4 (&acc)[4]) {
    float odd[4];  // (four chains: one of sixteen is waited for)
#pragma unroll
    for (int e = 0; e < 4; ++e) odd[e] = fmaf(acc[e][3], 0.0f, fmaf(acc[e][2], 0.0f, fmaf(acc[e][1], 0.0f, acc[e][0] * 0.0f)));
    const float all = (odd[0] + odd[1]) + (odd[2] + odd[3]);
    return __ballot(all != all) != 0;
}
// Sums that are not finite become those of the leading parts, if these are not either.
__device__ __forceinline__ void leading_kind(f32x4 &acc, const f32x4 &kind) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (!(fabsf(acc[i]) < __builtin_inff()) && !(fabsf(kind[i]) < __builtin_inff())) acc[i] = kind[i];
    __builtin_amdgcn_sched_barrier(0);  // (one after the other: what is rare takes few registers)
}

// Loads are never conditional: a lane without work of its own reads a place that exists (another row of the tile, the
// start of a row), so that all loads of a step are in flight together, and what it read meets a zero in the other operand or a
// result that is not stored.  (An infinity read that way belongs to the same token or adapter; the product with zero is then formed
// again without it, or it is cleared where the columns end.)
//
// How a kernel reaches the rows of its matrices:
//   ROWS_ALIGNED  16-byte vectors at 16-byte addresses, widths multiples of 8; the backward's kernels then step through the matrix they
//                 stream with byte offsets of 32 bits (matrices below 4 GiB: one addition per load)
//   ROWS_LOOSE    the same vectors at any address, the last one of a row moved back into it and shifted: odd widths, strides and
//                 starting points (511 tokens, H 1327, O 32,000, rank 32: 147 us a call entry by entry, 48 us so)
//   ROWS_SCALAR   entry by entry: rows of fewer than 8 entries
enum RowMode { ROWS_SCALAR = 0, ROWS_LOOSE = 1, ROWS_ALIGNED = 2 };
struct __attribute__((packed, aligned(2))) Loose16 { uint32_t w[4]; };
struct __attribute__((packed, aligned(2))) Loose8 { uint32_t w[2]; };
// The vector without its first d entries, 0 <= d < 8; zeros come in behind.
__device__ __forceinline__ uint4 drop_entries(const Loose16 &v, int d) {
    const uint64_t first = (uint64_t(v.w[1]) << 32) | v.w[0], second = (uint64_t(v.w[3]) << 32) | v.w[2];
    const uint64_t lo = d & 4 ? second : first, hi = d & 4 ? 0 : second;
    const int s = 16 * (d & 3);
    const uint64_t l = (lo >> s) | ((hi << 1) << (63 - s)), h = hi >> s;
    return make_uint4(uint32_t(l), uint32_t(l >> 32), uint32_t(h), uint32_t(h >> 32));
}
// Columns col .. col + 7 of a row of `width`; where they do not exist, other entries of the row, or zeros.
template <typename T, int MODE> __device__ __forceinline__ uint4 load8(const typename T::raw_t *row, int col, int width) {
    if constexpr (MODE == ROWS_ALIGNED) {
        return *reinterpret_cast<const uint4 *>(row + (col < width ? col : 0));
    } else if constexpr (MODE == ROWS_LOOSE) {
        const int c = col < width - 8 ? col : width - 8;
        return drop_entries(*reinterpret_cast<const Loose16 *>(row + c), (col - c) & 7);
    } else {
        uint32_t e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = row[col + j < width ? col + j : 0];
        return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
}
// The first n entries of a vector, zeros behind them.
__device__ __forceinline__ uint4 first_entries(const uint4 &v, int n) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = w[j] & ((2 * j < n ? 0xffffu : 0u) | (2 * j + 1 < n ? 0xffff0000u : 0u));
    return make_uint4(k[0], k[1], k[2], k[3]);
}
// load8 with zeros behind the row.
template <typename T, int MODE> __device__ __forceinline__ uint4 load8_zero(const typename T::raw_t *row, int col, int width) {
    const uint4 v = load8<T, MODE>(row, col, width);
    if constexpr (MODE == ROWS_ALIGNED) return col < width ? v : make_uint4(0, 0, 0, 0);
    else return first_entries(v, width - col);
}
// Columns col .. col + 7 of row `row` of a dense matrix [rows, width] of at least 8 entries, whose rows may be shorter than that;
// what lies behind the row is zero, or the row's own.
template <typename T, int MODE>
__device__ __forceinline__ uint4 dense_load8(const typename T::raw_t *matrix, int row, int rows, int col, int width) {
    if constexpr (MODE == ROWS_LOOSE) {
        const int64_t at = int64_t(row) * width + col, last = int64_t(rows) * width - 8;
        const int64_t from = at < last ? at : last;
        return first_entries(drop_entries(*reinterpret_cast<const Loose16 *>(matrix + from), int(at - from) & 7), width - col);
    } else {
        return load8<T, MODE>(matrix + int64_t(row) * width, col, width);
    }
}
template <typename T, int MODE> __device__ __forceinline__ uint2 load4(const typename T::raw_t *row, int col, int width) {
    if constexpr (MODE == ROWS_ALIGNED) {
        return *reinterpret_cast<const uint2 *>(row + (col < width ? col : 0));
    } else if constexpr (MODE == ROWS_LOOSE) {
        const int c = col < width - 4 ? col : width - 4;
        const Loose8 v = *reinterpret_cast<const Loose8 *>(row + c);
        const uint64_t l = ((uint64_t(v.w[1]) << 32) | v.w[0]) >> (16 * ((col - c) & 3));
        return make_uint2(uint32_t(l), uint32_t(l >> 32));
    } else {
        uint32_t e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = row[col + j < width ? col + j : 0];
        return make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
    }
}

// Rows of a streamed matrix, by byte offset.
template <int MODE> using row_offset_t = std::conditional_t<MODE == ROWS_ALIGNED, uint32_t, int64_t>;
template <int MODE> __device__ __forceinline__ row_offset_t<MODE> row_offset(int token, int64_t stride) {
    return row_offset_t<MODE>(token) * row_offset_t<MODE>(stride * 2);
}
template <typename T, int MODE> __device__ __forceinline__ const typename T::raw_t *row_at(const void *base, row_offset_t<MODE> at) {
    return reinterpret_cast<const typename T::raw_t *>(static_cast<const char *>(base) + at);
}
// Columns of a lane that stay the same for every row of a kernel: clamped to the row once where vectors are aligned.
template <int MODE> __device__ __forceinline__ int lane_column(int col, int width) { return MODE != ROWS_ALIGNED || col < width ? col : 0; }
template <typename T, int MODE> __device__ __forceinline__ uint2 row_load4(const void *base, row_offset_t<MODE> at, int col, int width) {
    if constexpr (MODE == ROWS_ALIGNED) return *reinterpret_cast<const uint2 *>(row_at<T, MODE>(base, at + row_offset_t<MODE>(col * 2)));
    else return load4<T, MODE>(row_at<T, MODE>(base, at), col, width);
}
template <typename T, int MODE> __device__ __forceinline__ uint4 row_load8(const void *base, row_offset_t<MODE> at, int col, int width) {
    if constexpr (MODE == ROWS_ALIGNED) return *reinterpret_cast<const uint4 *>(row_at<T, MODE>(base, at + row_offset_t<MODE>(col * 2)));
    else return load8<T, MODE>(row_at<T, MODE>(base, at), col, width);
}
// Eight rows of four columns -> the four fragments e whose contraction index is the row: column e of each.
__device__ __forceinline__ void transpose(const uint2 (&w)[8], uint4 (&frag)[4]) {
    uint32_t f[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[0][j] = __builtin_amdgcn_perm(w[2 * j + 1].x, w[2 * j].x, 0x05040100u);
        f[1][j] = __builtin_amdgcn_perm(w[2 * j + 1].x, w[2 * j].x, 0x07060302u);
        f[2][j] = __builtin_amdgcn_perm(w[2 * j + 1].y, w[2 * j].y, 0x05040100u);
        f[3][j] = __builtin_amdgcn_perm(w[2 * j + 1].y, w[2 * j].y, 0x07060302u);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) frag[e] = make_uint4(f[e][0], f[e][1], f[e][2], f[e][3]);
}

template <typename T> __device__ __forceinline__ typename T::raw_t narrow(float v) {
    if constexpr (T::kDtype == KA_DTYPE_BF16) return __builtin_bit_cast(uint16_t, __bf16(v));
    else return __builtin_bit_cast(uint16_t, _Float16(v));
}

// The sixteen results a lane holds for one token after four products e: columns first .. + 7 and first + 32 .. + 7, so that the
// four quads of a wavefront reach 64 contiguous bytes of a row with every access.  Which product and row they come from:
//   BY_HALF   MFMA row m of product e is column 32 (e / 2) + 8 (m / 4) + 4 (e % 2) + m % 4   (sixteen rows of B per load: four runs
//             of four)
//   BY_ROW    MFMA row m of product e is column permuted(m) + e                              (four columns of A per load)
// out = base + acc, rounded once; the base is loaded ahead of the products.
enum ColumnMap { BY_HALF, BY_ROW };
__device__ __forceinline__ int permuted(int m) { return (m & 2) * 16 + (m >> 2) * 8 + (m & 1) * 4; }
template <typename T, int MODE, int MAP> struct BaseRow {
    uint4 v[2];
    __device__ __forceinline__ void load(const void *base, int64_t row, int first, int width) {
        const typename T::raw_t *p = static_cast<const typename T::raw_t *>(base) + row;
#pragma unroll
        for (int h = 0; h < 2; ++h) v[h] = base != nullptr ? load8<T, MODE>(p, first + 32 * h, width) : make_uint4(0, 0, 0, 0);
    }
    static __device__ __forceinline__ float result(const f32x4 (&acc)[4], int h, int j) {
        return MAP == BY_HALF ? acc[2 * h + j / 4][j & 3] : acc[j & 3][2 * h + j / 4];
    }
    __device__ __forceinline__ void store(typename T::raw_t *out, int first, int width, const f32x4 (&acc)[4]) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = first + 32 * h;
            float b[8];
            T::unpack(v[h], b);
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v0 = b[2 * j] + result(acc, h, 2 * j), v1 = b[2 * j + 1] + result(acc, h, 2 * j + 1);
                w[j] = uint32_t(narrow<T>(v0)) | uint32_t(narrow<T>(v1)) << 16;
            }
            if constexpr (MODE == ROWS_ALIGNED) {
                if (c < width) *reinterpret_cast<uint4 *>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
            } else if (MODE == ROWS_LOOSE && c + 8 <= width) {
                *reinterpret_cast<Loose16 *>(out + c) = Loose16{{w[0], w[1], w[2], w[3]}};
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < width) out[c + j] = typename T::raw_t(w[j / 2] >> (16 * (j & 1)));
            }
        }
    }
};

// A barrier that orders LDS only: loads in flight stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Where R <= 16 one product of 32 holds the high parts of u in its first half and the low ones in its second.
template <int RP> struct Steps { static constexpr int kCount = RP <= 16 ? 1 : RP / 32; };

// first + part[0] + part[step] + ..., added in that order; U of them requested together (those that exist: the rest read the first).
template <int U> __device__ __forceinline__ float add_some(float sum, const float *__restrict__ part, int count, int64_t step) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = part[int64_t(u < count ? u : 0) * step];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < count) sum += v[u];
    return sum;
}
__device__ __forceinline__ float add_parts(float first, const float *__restrict__ part, int parts, int64_t step) {
    float sum = first;
    int q = 0;
    for (; q + 32 <= parts; q += 32) sum = add_some<32>(sum, part + int64_t(q) * step, 32, step);
    for (; q < parts; q += 8) sum = add_some<8>(sum, part + int64_t(q) * step, parts - q, step);
    return sum;
}

// ---------------------------------------------------------------------------
// lora_shrink: u = s x A^T.  H is cut into segments of 1024; inside one the wavefronts take two of every eight steps of 32 and
// are added in their order, and the segments are added in theirs: by one workgroup (grid (1, tiles)), or by the reader of one
// partial result per segment (grid (segments, tiles)) where the tiles alone would leave CUs idle.  The bits of a token's u
// do not depend on which of the two runs, nor on the other tokens.
// ONE: a call of few tokens, one per workgroup, which need no plan; one more workgroup makes it for the kernel behind.
// Bound by the reads of x and, with many adapters, of A: 64 tokens over 16 adapters of rank 16, H 4096: 5.8 us; 5003 tokens, rank 64
// (fp16, 41 MB): 22 us, 1.9 TB/s (data that no cache holds, here and below).
// ---------------------------------------------------------------------------
constexpr int SEG_STEPS = 32;  // steps of 32 per segment
struct ShrinkArgs {
    const void *x, *a;
    int64_t x_stride;
    const int64_t *ids;
    const float *scaling;
    float scale;
    int32_t n, h, r, s, segments, split;
    float *out;  // [N, R] scaled, or with `split` [segments, N, R]
    LoraPlan plan;
};
template <typename T, int RP, int MODE, bool ONE>
__global__ __launch_bounds__(THREADS) void lora_shrink(ShrinkArgs p) {
    constexpr int RF = RP / 16, SUBS = ONE ? 1 : FWD_SUBS;
    __shared__ union {
        f32x4 part[WAVES][SUBS * 16][4];  // [wave][token][rank / 4] of one group of sixteen ranks
        std::conditional_t<ONE, PlanShared<THREADS>, int> plan;
    } sh;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, quad = lane >> 4;
    LoraTile tile;
    if constexpr (ONE) {
        if (int(blockIdx.y) == p.n) {
            if (blockIdx.x == 0) make_plan(sh.plan, p.ids, p.n, p.s, 1, p.plan);
            return;
        }
        const int64_t id = p.ids[blockIdx.y];
        tile.adapter = id >= 0 && id < p.s ? int(id) : -1;
        tile.count = 1;
    } else {
        if (int(blockIdx.y) >= *p.plan.list[0].count) return;
        tile = p.plan.list[0].tiles[blockIdx.y];
    }
    auto token_of = [&](int i) { return ONE ? int(blockIdx.y) : p.plan.order[tile.start + (i < tile.count ? i : 0)]; };
    const int mine = tid / 4, mine_q = tid & 3;  // the thread adds up four ranks of token `mine` of the tile
    f32x4 sum[RF];
#pragma unroll
    for (int f = 0; f < RF; ++f) sum[f] = f32x4{0, 0, 0, 0};
    if (tile.adapter >= 0) {
        const typename T::raw_t *rows[SUBS];
#pragma unroll
        for (int s = 0; s < SUBS; ++s) rows[s] = static_cast<const typename T::raw_t *>(p.x) + int64_t(token_of(s * 16 + col)) * p.x_stride;
        const typename T::raw_t *aw = static_cast<const typename T::raw_t *>(p.a) + int64_t(tile.adapter) * p.r * p.h;
        const int steps = (p.h + 31) / 32;
        const int seg0 = p.split ? int(blockIdx.x) : 0, seg1 = p.split ? seg0 + 1 : p.segments;
        for (int seg = seg0; seg < seg1; ++seg) {
            f32x4 acc[RF][SUBS];
#pragma unroll
            for (int f = 0; f < RF; ++f)
#pragma unroll
                for (int s = 0; s < SUBS; ++s) acc[f][s] = f32x4{0, 0, 0, 0};
            const int end = (seg + 1) * SEG_STEPS < steps ? (seg + 1) * SEG_STEPS : steps;
            // a wavefront takes two neighbouring steps of every eight: whole 128-byte lines of the rows
#pragma unroll(RP <= 32 ? 2 : 1)
            for (int st = seg * SEG_STEPS + 2 * wave; st < end; st += 2 * WAVES) {
                uint4 fa[2][RF], fx[2][SUBS];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int k = (st + t) * 32 + 8 * quad;
#pragma unroll
                    for (int f = 0; f < RF; ++f) fa[t][f] = load8_zero<T, MODE>(aw + int64_t(f * 16 + col < p.r ? f * 16 + col : 0) * p.h, k, p.h);
#pragma unroll
                    for (int s = 0; s < SUBS; ++s) fx[t][s] = load8<T, MODE>(rows[s], k, p.h);
                }
                if ((st + 2) * 32 > p.h) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int s = 0; s < SUBS; ++s) fx[t][s] = first_entries(fx[t][s], p.h - (st + t) * 32 - 8 * quad);
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int f = 0; f < RF; ++f)
#pragma unroll
                        for (int s = 0; s < SUBS; ++s) acc[f][s] = mfma<T>(fa[t][f], fx[t][s], acc[f][s]);
            }
#pragma unroll
            for (int f = 0; f < RF; ++f) {
                __syncthreads();  // the previous parts are read
#pragma unroll
                for (int s = 0; s < SUBS; ++s) sh.part[wave][s * 16 + col][quad] = acc[f][s];
                __syncthreads();
                if (mine < SUBS * 16) {
                    f32x4 v = sh.part[0][mine][mine_q];
#pragma unroll
                    for (int w = 1; w < WAVES; ++w) v += sh.part[w][mine][mine_q];
                    sum[f] += v;
                }
            }
        }
    }
    if (mine >= tile.count) return;
    const float scale = tile.adapter < 0 ? 0.0f : (p.split ? 1.0f : (p.scaling != nullptr ? p.scaling[tile.adapter] : p.scale));
    float *out = p.out + (p.split ? int64_t(blockIdx.x) * p.n * p.r : 0) + int64_t(token_of(mine)) * p.r;
#pragma unroll
    for (int f = 0; f < RF; ++f) {
        const int r0 = f * 16 + mine_q * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (r0 + j < p.r) out[r0 + j] = tile.adapter < 0 ? 0.0f : sum[f][j] * scale;
    }
}

// out[n, r] = s_a sum over the parts, in order; 0 for tokens without an adapter.
__global__ __launch_bounds__(THREADS) void lora_fold_rows(const float *__restrict__ part, int parts, int64_t n, int r,
                                                          const int64_t *__restrict__ ids, int s, const float *__restrict__ scaling,
                                                          float scale, float *__restrict__ out) {
    const int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x;
    if (i >= n * r) return;
    const int64_t a = ids[i / r];
    float v = 0.0f;
    if (a >= 0 && a < s) v = add_parts(0.0f, part + i, parts, n * r) * (scaling != nullptr ? scaling[a] : scale);
    out[i] = v;
}

// ---------------------------------------------------------------------------
// lora_expand: grid (blocks of O, tiles).  y = base + u B^T for the tokens of a tile.
//
// u enters as fragments (column = token, contraction index = rank) of its high and low bf16 parts, 17 bits of every entry.
// They come packed from lora_pack_rows, or in calls of few tokens (PARTS) from the segments of lora_shrink.
// Bound by memory, base in and out through: 64 tokens x 128,256 outputs, 16 adapters of rank 16 (99 MB): 26 us, 3.9 TB/s, fp16 29;
// 5003 tokens x 4096, rank 64 (82 MB): 29 us, 2.8 TB/s, fp16 33.  Tiles of 32 tokens: at 64 an adapter with a few tokens left half of the
// products empty and the registers let two workgroups reside instead of four.  The builds for aligned rows hold everything in
// registers; those for any address spill up to 10 of them.
// ---------------------------------------------------------------------------
template <int RP> struct RowFragments {  // of 32 tokens, in uint4: [group of 16][step][high, low][lane]
    static constexpr int kSteps = Steps<RP>::kCount, kParts = RP <= 16 ? 1 : 2;
    static constexpr int kTotal = FWD_SUBS * kSteps * kParts * kWave;
};
// The fragment of a group and step (both parts) from eight values of u a lane.
template <int RP> __device__ __forceinline__ void row_fragment(const float (&v)[8], uint4 *out, int lane) {
    uint4 hl[2];
    split<2>(v, hl);
    if (RP <= 16) {
        out[lane] = choose((lane >> 4) < 2, hl[0], hl[1]);
    } else {
        out[lane] = hl[0];
        out[kWave + lane] = hl[1];
    }
}

// grid (tiles): u of a tile's tokens from `parts` segments, added in order and scaled; also to out_shrunk.
struct PackRowsArgs {
    const float *part;
    float *out_shrunk;  // may be null
    const float *scaling;
    float scale;
    int32_t parts, scaled, r;
    int64_t n;
    uint4 *out;
    LoraPlan plan;
};
template <int RP>
__global__ __launch_bounds__(THREADS) void lora_pack_rows(PackRowsArgs p) {
    constexpr int KS = Steps<RP>::kCount, LD = RP + 1;
    __shared__ float v[FWD_TILE * LD];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, quad = lane >> 4;
    const LoraTile tile = p.plan.list[0].tiles[blockIdx.x];
    if (int(blockIdx.x) >= *p.plan.list[0].count) return;
    const float scale = tile.adapter < 0 ? 0.0f : (p.scaling != nullptr ? p.scaling[tile.adapter] : p.scale);
    for (int i = tid; i < FWD_TILE * RP; i += THREADS) {
        const int t = i / RP, rank = i % RP;
        float x = 0.0f;
        if (t < tile.count && rank < p.r) {
            const int64_t at = int64_t(p.plan.order[tile.start + t]) * p.r + rank;
            if (tile.adapter >= 0) {
                x = add_parts(0.0f, p.part + at, p.parts, p.n * p.r);
                if (p.scaled) x *= scale;
            }
            if (p.out_shrunk != nullptr) p.out_shrunk[at] = x;
        }
        v[t * LD + rank] = x;
    }
    __syncthreads();
    uint4 *out = p.out + int64_t(blockIdx.x) * RowFragments<RP>::kTotal;
    for (int q = wave; q < FWD_SUBS * KS; q += WAVES) {
        const int s = q / KS, ks = q % KS;
        const int r0 = RP <= 16 ? 8 * (quad & 1) : 32 * ks + 8 * quad;
        const float *row = v + (16 * s + col) * LD;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = row[r0 + j];
        row_fragment<RP>(x, out + q * RowFragments<RP>::kParts * kWave, lane);
    }
}

struct ExpandArgs {
    const void *base, *b;
    void *out;
    int64_t base_stride, out_stride;
    const uint4 *packed;  // RowFragments per tile
    const float *u;       // PARTS: [parts, N, R], the segments before the scaling
    float *out_shrunk;    // PARTS: u, written by the first block of outputs of every tile; may be null
    const float *scaling;
    float scale;
    int64_t n;
    int32_t parts, o, r, groups, in_place;  // groups: of 64 outputs per wavefront
    LoraPlan plan;
};
template <typename T, int RP, int MODE, bool PARTS>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(RP <= 32 ? 4 : 2))) void lora_expand(ExpandArgs p) {
    constexpr int KS = Steps<RP>::kCount, HL = RP <= 16 ? 1 : 2, NP = Parts<T>::kCount;
    __shared__ uint4 uf[PARTS ? FWD_SUBS * KS * HL * kWave : 1];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, quad = lane >> 4;
    const LoraTile tile = p.plan.list[0].tiles[blockIdx.y];  // (in the list's memory also where there is no such tile)
    if (int(blockIdx.y) >= *p.plan.list[0].count) return;
    const bool shrunk_out = PARTS && p.out_shrunk != nullptr && blockIdx.x == 0;
    if (tile.adapter < 0 && p.in_place && !shrunk_out) return;
    const bool two = tile.count > 16;
    int token[FWD_SUBS];  // (a column without a token: the tile's first)
    bool live[FWD_SUBS];
#pragma unroll
    for (int s = 0; s < FWD_SUBS; ++s) {
        live[s] = s * 16 + col < tile.count;
        token[s] = p.plan.order[tile.start + (live[s] ? s * 16 + col : 0)];
    }
    const typename T::raw_t *bw = static_cast<const typename T::raw_t *>(p.b) + int64_t(tile.adapter < 0 ? 0 : tile.adapter) * p.o * p.r;
    struct Stage {
        BaseRow<T, MODE, BY_HALF> row[FWD_SUBS];
        uint4 b[KS][4];
    };
    auto first_of = [&](int g) { return ((int(blockIdx.x) * p.groups + g) * WAVES + wave) * 64; };
    auto b_fragment = [&](int o0, int ks, int e) {
        const int o = o0 + 32 * (e / 2) + 8 * (col / 4) + 4 * (e & 1) + (col & 3);
        return dense_load8<T, MODE>(bw, o < p.o ? o : 0, p.o, RP <= 16 ? 8 * (quad & 1) : 32 * ks + 8 * quad, p.r);
    };
    auto request = [&](int g, Stage &st) {
        const int o0 = first_of(g) < p.o ? first_of(g) : 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.b[ks][e] = b_fragment(o0, ks, e);
        st.row[0].load(p.base, token[0] * p.base_stride, o0 + 8 * quad, p.o);
        if (two) st.row[1].load(p.base, token[1] * p.base_stride, o0 + 8 * quad, p.o);
    };
    Stage even;
    request(0, even);
    uint4 fu[PARTS ? 1 : FWD_SUBS][KS][HL];
    if constexpr (!PARTS) {
        const uint4 *packed = p.packed + int64_t(blockIdx.y) * RowFragments<RP>::kTotal;
#pragma unroll
        for (int s = 0; s < FWD_SUBS; ++s)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int k = 0; k < HL; ++k) fu[s][ks][k] = packed[((s * KS + ks) * HL + k) * kWave + lane];
    } else {
        const float scale = tile.adapter < 0 ? 0.0f : (p.scaling != nullptr ? p.scaling[tile.adapter] : p.scale);
        for (int q = wave; q < FWD_SUBS * KS; q += WAVES) {
            const int s = q % FWD_SUBS, ks = q / FWD_SUBS;
            const bool mine = (s == 0 ? live[0] : live[1]) && tile.adapter >= 0;
            const int64_t row = int64_t(s == 0 ? token[0] : token[1]) * p.r;
            auto load_u = [&](int r0, float (&v)[8]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = 0.0f;
                for (int part = 0; part < p.parts; part += 4) {
                    float x[4][8];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const float *at = p.u + (part + t < p.parts ? part + t : part) * p.n * p.r + row;
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[t][j] = at[r0 + j < p.r ? r0 + j : 0];
                    }
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        if (part + t < p.parts) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] += x[t][j];
                        }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = mine && r0 + j < p.r ? v[j] * scale : 0.0f;
            };
            const int r0 = RP <= 16 ? 8 * (quad & 1) : 32 * ks + 8 * quad;
            float own[8];
            load_u(r0, own);
            if (shrunk_out && (s == 0 ? live[0] : live[1]) && (RP > 16 || quad < 2)) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (r0 + j < p.r) p.out_shrunk[row + r0 + j] = own[j];
            }
            row_fragment<RP>(own, uf + (s * KS + ks) * HL * kWave, lane);
        }
        lds_barrier();
    }
    if (tile.adapter < 0 && p.in_place) return;
    typename T::raw_t *out = static_cast<typename T::raw_t *>(p.out);
    // Groups whose products run side by side: both for fp16, so that the parts of a fragment of B are made once and kept for no longer.
    constexpr int SIDE = NP == 1 ? 1 : FWD_SUBS;
    auto finish = [&](int g, const Stage &st) {
        const int o0 = first_of(g);
        if (o0 >= p.o) return;
#pragma unroll
        for (int s0 = 0; s0 < FWD_SUBS; s0 += SIDE) {
            if (s0 == 1 && !two) continue;
            f32x4 acc[SIDE][4];
#pragma unroll
            for (int s = 0; s < SIDE; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[s][e] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint4 f[SIDE][HL];
#pragma unroll
                for (int s = 0; s < SIDE; ++s)
#pragma unroll
                    for (int k = 0; k < HL; ++k) {
                        if constexpr (PARTS) f[s][k] = uf[(((s0 + s) * KS + ks) * HL + k) * kWave + lane];
                        else f[s][k] = fu[s0 + s][ks][k];
                    }
                if constexpr (NP == 1) {
#pragma unroll
                    for (int k = 0; k < HL; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[0][e] = mfma<Bf16>(st.b[ks][e], f[0][k], acc[0][e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint4 part[NP];
                        as_bf16<T>(st.b[ks][e], part);
#pragma unroll
                        for (int q = NP - 1; q >= 0; --q)
#pragma unroll
                            for (int s = 0; s < SIDE; ++s)
#pragma unroll
                                for (int k = HL - 1; k >= 0; --k) acc[s][e] = mfma<Bf16>(part[q], f[s][k], acc[s][e]);
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < SIDE; ++s) {
                if (tile.adapter >= 0 && any_odd(acc[s])) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f32x4 kind = {0, 0, 0, 0};
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            // (ranks of this lane; with R <= 16 the second half of the lanes holds low parts)
                            const int ranks = RP <= 16 ? (quad < 2 ? p.r - 8 * quad : 0) : p.r - 32 * ks - 8 * quad;
                            uint4 f, part[NP];
                            if constexpr (PARTS) f = uf[((s0 + s) * KS + ks) * HL * kWave + lane];
                            else f = p.packed[int64_t(blockIdx.y) * RowFragments<RP>::kTotal + ((s0 + s) * KS + ks) * HL * kWave + lane];
                            as_bf16<T>(b_fragment(o0, ks, e), part);  // (read again, so that the products above need not keep it)
                            kind = mfma<Bf16>(first_entries(part[0], ranks), first_entries(f, ranks), kind);
                        }
                        leading_kind(acc[s][e], kind);
                    }
                }
                // (0 times an infinity of the rows that were read in their place would not be 0)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[s][e][i] = tile.adapter >= 0 ? acc[s][e][i] : 0.0f;
                if (live[s0 + s]) st.row[s0 + s].store(out + token[s0 + s] * p.out_stride, o0 + 8 * quad, p.o, acc[s]);
            }
        }
    };
    // Two stages of outputs where the registers of four wavefronts per SIMD hold them.  fp16 keeps the parts of a fragment of B and both
    // groups' sums beside them and would spill; us a call with two stages and with one: rank 16, 64 tokens x 128,256 outputs 42.6 / 39.3,
    // 8192 x 4096 94 / 83; rank 32, 5003 x 4096 75 / 67.
    if constexpr (RP <= 32 && NP == 1) {
        // what the next 64 outputs need is requested before the products of the present ones
        Stage odd;
        for (int g = 0; g < p.groups; g += 2) {
            if (g + 1 < p.groups) request(g + 1, odd);
            finish(g, even);
            if (g + 1 < p.groups) {
                if (g + 2 < p.groups) request(g + 2, even);
                finish(g + 1, odd);
            }
        }
    } else {
        for (int g = 0; g < p.groups; ++g) {
            if (g > 0) request(g, even);
            finish(g, even);
        }
    }
}

// ---------------------------------------------------------------------------
// lora_fold_parts: grid (elements / 256, groups).  Sums of 32 neighbouring partial results, all requested together, where there
// are so many that the few workgroups of lora_pack would wait for them one after the other (512 tokens, rank 128, 501 parts: 235 us in
// lora_pack alone, 21 + 10 us so).
// ---------------------------------------------------------------------------
constexpr int FOLD_PARTS = 32;
__global__ __launch_bounds__(THREADS) void lora_fold_parts(const float *__restrict__ part, int parts, int64_t elements, float *__restrict__ out) {
    const int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x;
    if (i >= elements) return;
    const int first = int(blockIdx.y) * FOLD_PARTS;
    const float *at = part + int64_t(first) * elements + i;
    out[int64_t(blockIdx.y) * elements + i] = add_some<FOLD_PARTS>(0.0f, at, parts - first, elements);
}

// ---------------------------------------------------------------------------
// lora_pack: grid (tiles of the first list).  u, or the sum of the partial results of dy B times s_a, for every 32 tokens of an
// adapter in the layout and precision the matrix cores take it in, so that the workgroups of the two passes over the data load
// fragments and split nothing:
//   columns  [rank group][part 0 .. 2][lane]   contraction index = token, three bf16 parts (24 bits)
//   rows     [group of 16 tokens][step][high, low][lane]   contraction index = rank (only for dy B)
// The chunk of 32 tokens that starts at position i of `order`, in adapter a, is chunk i / 32 + a.
// ---------------------------------------------------------------------------
template <int RP> struct Packed {
    static constexpr int kColumns = RP / 16 * 3 * kWave;                               // in uint4
    static constexpr int kRows = 2 * Steps<RP>::kCount * (RP <= 16 ? 1 : 2) * kWave;
};
struct PackArgs {
    const float *part;  // [parts, N, R]
    int32_t parts, r, rows;
    int64_t n;
    const float *scaling;  // null: scale
    float scale;
    int32_t scaled;
    uint4 *out;
    LoraPlan plan;
};
template <int RP>
__global__ __launch_bounds__(THREADS) void lora_pack(PackArgs p) {
    constexpr int RF = RP / 16, KS = Steps<RP>::kCount, HL = RP <= 16 ? 1 : 2, LD = RP + 1;
    __shared__ float v[32 * LD];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, quad = lane >> 4;
    if (int(blockIdx.y) >= *p.plan.list[0].count) return;
    const LoraTile tile = p.plan.list[0].tiles[blockIdx.y];
    const int c = int(blockIdx.x) * 32;
    if (tile.adapter < 0 || c >= tile.count) return;
    const float scale = !p.scaled ? 1.0f : (p.scaling != nullptr ? p.scaling[tile.adapter] : p.scale);
    for (int i = tid; i < 32 * RP; i += THREADS) {
        const int t = i / RP, rank = i % RP;
        float x = 0.0f;
        if (c + t < tile.count && rank < p.r) {
            const float *at = p.part + int64_t(p.plan.order[tile.start + c + t]) * p.r + rank;
            x = add_parts(0.0f, at, p.parts, p.n * p.r) * scale;
        }
        v[t * LD + rank] = x;
    }
    __syncthreads();
    uint4 *out = p.out + int64_t((tile.start + c) / 32 + tile.adapter) * (Packed<RP>::kColumns + (p.rows ? Packed<RP>::kRows : 0));
    for (int f = wave; f < RF; f += WAVES) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[(8 * quad + j) * LD + f * 16 + col];
        uint4 part[3];
        split<3>(x, part);
#pragma unroll
        for (int k = 0; k < 3; ++k) out[(f * 3 + k) * kWave + lane] = part[k];
    }
    if (!p.rows) return;
    out += Packed<RP>::kColumns;
    for (int q = wave; q < 2 * KS; q += WAVES) {
        const int s = q / KS, ks = q % KS;
        const int r0 = RP <= 16 ? 8 * (quad & 1) : 32 * ks + 8 * quad;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[(16 * s + col) * LD + r0 + j];
        uint4 hl[2];
        split<2>(x, hl);
        if (RP <= 16) {
            out[q * kWave + lane] = choose(quad < 2, hl[0], hl[1]);
        } else {
            out[(q * HL) * kWave + lane] = hl[0];
            out[(q * HL + HL - 1) * kWave + lane] = hl[1];
        }
    }
}

// ---------------------------------------------------------------------------
// lora_bwd_out: grid (blocks of O, tiles).  One pass over dy: the tile's part of dB, and dy B over the block's outputs.
// A wavefront owns 64 G outputs; per 32 tokens it reads them twice (once from HBM, once from cache): transposed for dB, as
// they are for dy B.  What a step needs from HBM is requested a step ahead (two steps ahead measured slower: 301 -> 335 us below).
// Bound by the wait for those rows with one wavefront per SIMD (rank 16 with G = 4, rank 128; two at rank 64): 4096 tokens x 128,256
// outputs, rank 16 (1.05 GB): 297 us, 3.5 TB/s; 2048 x 4096: 12 us; rank 64, 1024 x 128,256: 166 us; rank 128, 512 x 128,256: 180 us, of
// which the three products of the gradient's split take about 40.
// ---------------------------------------------------------------------------
struct BwdOutArgs {
    const void *dy, *b;
    int64_t dy_stride;
    const uint4 *u;       // packed columns
    int32_t n, o, r;
    float *db, *db_part;  // [S, O, R], [slots, O, R]
    float *du_part;       // [blocks, N, R]
    LoraPlan plan;
};
// The tile's tokens into LDS, the last one repeated up to a multiple of 32.
__device__ __forceinline__ void load_tokens(const int32_t *order, const LoraTile &tile, int32_t *tokens) {
    for (int i = threadIdx.x; i < (tile.count + 31) / 32 * 32; i += THREADS) tokens[i] = order[tile.start + (i < tile.count ? i : tile.count - 1)];
}
__device__ __forceinline__ void eight_tokens(const int32_t *tokens, int32_t (&t)[8]) {
    const int4 a = *reinterpret_cast<const int4 *>(tokens), b = *reinterpret_cast<const int4 *>(tokens + 4);
    t[0] = a.x; t[1] = a.y; t[2] = a.z; t[3] = a.w;
    t[4] = b.x; t[5] = b.y; t[6] = b.z; t[7] = b.w;
}
// acc += data^T v for one column group: parts of the data times parts of v, small products first
template <typename T> __device__ __forceinline__ f32x4 outer(const uint4 (&data)[Parts<T>::kCount], const uint4 (&v)[3], f32x4 acc) {
    if constexpr (Parts<T>::kCount == 2) {
        acc = mfma<Bf16>(data[1], v[1], acc);
        acc = mfma<Bf16>(data[1], v[0], acc);
    }
    acc = mfma<Bf16>(data[0], v[2], acc);
    acc = mfma<Bf16>(data[0], v[1], acc);
    return mfma<Bf16>(data[0], v[0], acc);
}
// What a gradient's sums are by their leading parts: data(c, j) loads four columns of token 8 quad + j of the 32 at c, `v` the leading parts of
// the other operand for the first 32 tokens, `step` further for the next.
template <typename T, typename F>
__device__ __forceinline__ void gradient_kind(f32x4 (&acc)[4], int count, const uint4 *v, int step, F &&data) {
    const int quad = (int(threadIdx.x) & (kWave - 1)) >> 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f32x4 kind = {0, 0, 0, 0};
#pragma unroll 1
        for (int c = 0; c < count; c += 32) {
            uint2 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = c + 8 * quad + j < count ? data(c, j) : make_uint2(0, 0);
            uint4 frag[4], part[Parts<T>::kCount];
            transpose(w, frag);
            as_bf16<T>(frag[e], part);
            kind = mfma<Bf16>(part[0], v[int64_t(c / 32) * step], kind);
        }
        leading_kind(acc[e], kind);
    }
}
template <typename T, int RP, int G, int MODE>
__global__ __launch_bounds__(THREADS) void lora_bwd_out(BwdOutArgs p) {
    constexpr int RF = RP / 16, NP = Parts<T>::kCount;
    constexpr int RED = RF < 4 ? RF : 4;  // groups of sixteen ranks that cross the wavefronts at a time
    __shared__ __attribute__((aligned(16))) int32_t tokens[BWD_TILE_MAX];
    __shared__ f32x4 red[WAVES][32][RED * 4];
    constexpr int US = RF * 3 * kWave, US_PER = (US + THREADS - 1) / THREADS;
    __shared__ u32x4 us[US];  // fragments of u for the step, the same for every wavefront
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, quad = lane >> 4;
    if (int(blockIdx.y) >= *p.plan.list[0].count) return;
    const LoraTile tile = p.plan.list[0].tiles[blockIdx.y];
    if (tile.adapter < 0) return;
    load_tokens(p.plan.order, tile, tokens);
    const typename T::raw_t *bw = static_cast<const typename T::raw_t *>(p.b) + int64_t(tile.adapter) * p.o * p.r;
    const int o0 = (int(blockIdx.x) * WAVES + wave) * 64 * G;
    const bool cut_short = (int(blockIdx.x) + 1) * WAVES * 64 * G > p.o;  // of the workgroup's outputs some do not exist
    // B^T fragments: row = rank, contraction index = output
    uint4 fb[G][2][RF];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int f = 0; f < RF; ++f) {
                uint32_t w[4];
                const int rank = f * 16 + col < p.r ? f * 16 + col : 0, o = o0 + g * 64 + ks * 32 + 8 * quad;
                uint32_t e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = bw[int64_t(o + j < p.o ? o + j : 0) * p.r + rank];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (o + 2 * j < p.o ? e[2 * j] : 0u) | (o + 2 * j + 1 < p.o ? e[2 * j + 1] << 16 : 0u);
                fb[g][ks][f] = make_uint4(w[0], w[1], w[2], w[3]);
            }
    f32x4 acc[G][RF][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int f = 0; f < RF; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[g][f][e] = f32x4{0, 0, 0, 0};
    __syncthreads();
    int col4[G], col8[G][2];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        col4[g] = lane_column<MODE>(o0 + g * 64 + 4 * col, p.o);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) col8[g][ks] = lane_column<MODE>(o0 + g * 64 + ks * 32 + 8 * quad, p.o);
    }
    const u32x4 *const packed = reinterpret_cast<const u32x4 *>(p.u) + int64_t(tile.start / 32 + tile.adapter) * Packed<RP>::kColumns + tid;
    auto request = [&](int c, uint2 (&w)[G][8]) {
        int32_t tk[8];
        eight_tokens(tokens + c + 8 * quad, tk);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const row_offset_t<MODE> at = row_offset<MODE>(tk[j], p.dy_stride);
#pragma unroll
            for (int g = 0; g < G; ++g) w[g][j] = row_load4<T, MODE>(p.dy, at, col4[g], p.o);
        }
    };
    auto step = [&](int c, const uint2 (&w)[G][8], uint2 (&next)[G][8]) {
        // the step's own remaining loads first (they come from cache), then the next step's; none behind those, since loads are
        // waited for in their order
        uint4 fy[G][2][2];
        u32x4 next_u[US_PER];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const row_offset_t<MODE> at = row_offset<MODE>(tokens[c + 16 * s + col], p.dy_stride);
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) fy[g][ks][s] = row_load8<T, MODE>(p.dy, at, col8[g][ks], p.o);
        }
        const int then = c + 32 < tile.count ? c + 32 : c;
#pragma unroll
        for (int i = 0; i < US_PER; ++i) next_u[i] = packed[int64_t(then / 32) * Packed<RP>::kColumns + i * THREADS];
        request(then, next);
        f32x4 du[2][RF];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int f = 0; f < RF; ++f) du[s][f] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint4 frag[4], part[4][NP];
            transpose(w[g], frag);
#pragma unroll
            for (int e = 0; e < 4; ++e) as_bf16<T>(frag[e], part[e]);
#pragma unroll
            for (int f = 0; f < RF; ++f) {
                uint4 v[3];
#pragma unroll
                for (int k = 0; k < 3; ++k) v[k] = __builtin_bit_cast(uint4, us[(f * 3 + k) * kWave + lane]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[g][f][e] = outer<T>(part[e], v, acc[g][f][e]);
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int f = 0; f < RF; ++f) du[s][f] = mfma<T>(fb[g][ks][f], fy[g][ks][s], du[s][f]);
        }
        // dy B of the workgroup's outputs: the wavefronts' parts in their order
        lds_barrier();  // the previous sums and the step's u are read
#pragma unroll
        for (int i = 0; i < US_PER; ++i)
            if (i * THREADS + tid < US) us[i * THREADS + tid] = next_u[i];
#pragma unroll
        for (int f0 = 0; f0 < RF; f0 += RED) {
            if (f0 > 0) lds_barrier();
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int f = 0; f < RED; ++f) red[wave][16 * s + col][f * 4 + quad] = du[s][f0 + f];
            lds_barrier();
            for (int q = tid; q < 32 * RED * 4; q += THREADS) {
                const int i = q / (RED * 4), r4 = q % (RED * 4), r0 = f0 * 16 + r4 * 4;
                if (c + i < tile.count && r0 < p.r) {
                    f32x4 sum = red[0][i][r4];
#pragma unroll
                    for (int k = 1; k < WAVES; ++k) sum += red[k][i][r4];
                    if (cut_short && !(fabsf(sum[0] * 0.0f + sum[1] * 0.0f + sum[2] * 0.0f + sum[3] * 0.0f) < 1.0f)) {
                        // a lane behind the last output read another one, of which an infinity times 0 is no number: entry by entry
                        const typename T::raw_t *row = row_at<T, MODE>(p.dy, row_offset<MODE>(tokens[c + i], p.dy_stride));
                        sum = f32x4{0, 0, 0, 0};
#pragma unroll 1
                        for (int o = int(blockIdx.x) * WAVES * 64 * G; o < p.o; ++o)
#pragma unroll
                            for (int j = 0; j < 4; ++j) sum[j] += T::widen(row[o]) * T::widen(bw[int64_t(o) * p.r + (r0 + j < p.r ? r0 + j : r0)]);
                    }
                    float *out = p.du_part + (int64_t(blockIdx.x) * p.n + tokens[c + i]) * p.r + r0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (r0 + j < p.r) out[j] = sum[j];
                }
            }
        }
    };
    uint2 even[G][8], odd[G][8];
    {
        u32x4 first_u[US_PER];
#pragma unroll
        for (int i = 0; i < US_PER; ++i) first_u[i] = packed[i * THREADS];
        request(0, even);
#pragma unroll
        for (int i = 0; i < US_PER; ++i)
            if (i * THREADS + tid < US) us[i * THREADS + tid] = first_u[i];
        lds_barrier();
    }
    for (int c = 0; c < tile.count; c += 64) {
        step(c, even, odd);
        if (c + 32 >= tile.count) break;
        step(c + 32, odd, even);
    }
    // sums of tokens that are not finite, once more from the leading parts
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int f = 0; f < RF; ++f)
            if (any_odd(acc[g][f]))
                gradient_kind<T>(acc[g][f], tile.count, reinterpret_cast<const uint4 *>(packed) - tid + f * 3 * kWave + lane, Packed<RP>::kColumns,
                                 [&](int c, int j) {
                                     return row_load4<T, MODE>(p.dy, row_offset<MODE>(tokens[c + 8 * quad + j], p.dy_stride), col4[g], p.o);
                                 });
    float *db = tile.slot < 0 ? p.db + int64_t(tile.adapter) * p.o * p.r : p.db_part + int64_t(tile.slot) * p.o * p.r;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int f = 0; f < RF; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int o = o0 + g * 64 + 16 * quad + 4 * i + e, rank = f * 16 + col;
                    if (o < p.o && rank < p.r) db[int64_t(o) * p.r + rank] = acc[g][f][e][i];
                }
}

// ---------------------------------------------------------------------------
// lora_bwd_in: grid (blocks of H, tiles).  One pass over x: the tile's part of dA, and dx = dx_base + du A.  Bound by memory:
// 4096 tokens x 4096 (100 MB): 30 us, 3.3 TB/s; 2048 x 4096: 22 us.
// ---------------------------------------------------------------------------
struct BwdInArgs {
    const void *x, *a, *dx_base;
    void *dx;
    int64_t x_stride, dx_base_stride, dx_stride;
    const uint4 *du;      // packed columns and rows
    int32_t h, r;
    float *da, *da_part;  // [S, R, H], [slots, R, H]
    LoraPlan plan;
};
template <typename T, int RP, int MODE>
// (three wavefronts per SIMD at rank 16, as many as the hot loop alone would have: 2048 x 4096, fp16 57.6 us a call, with two 61.5)
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(RP <= 16 ? 3 : RP <= 32 ? 2 : 1))) void lora_bwd_in(BwdInArgs p) {
    constexpr int RF = RP / 16, KS = Steps<RP>::kCount, HL = RP <= 16 ? 1 : 2, NP = Parts<T>::kCount;
    __shared__ __attribute__((aligned(16))) int32_t tokens[BWD_TILE_MAX];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, col = lane & 15, quad = lane >> 4;
    if (int(blockIdx.y) >= *p.plan.list[1].count) return;
    const LoraTile tile = p.plan.list[1].tiles[blockIdx.y];
    load_tokens(p.plan.order, tile, tokens);
    __syncthreads();
    const int h0 = (int(blockIdx.x) * WAVES + wave) * 64;
    if (h0 >= p.h) return;  // (no barrier follows)
    const bool has = tile.adapter >= 0;
    const typename T::raw_t *aw = static_cast<const typename T::raw_t *>(p.a) + (has ? int64_t(tile.adapter) * p.r * p.h : 0);
    const int col4 = lane_column<MODE>(h0 + permuted(col), p.h), out_col = h0 + 8 * quad;
    const uint4 *const packed = p.du + int64_t(tile.start / 32 + (has ? tile.adapter : 0)) * (Packed<RP>::kColumns + Packed<RP>::kRows) + lane;
    // A fragments: row permuted(m) + e = input, contraction index = rank
    uint4 fa[KS][4][NP];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        uint2 w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int rank = (RP <= 16 ? 8 * (quad & 1) : 32 * ks + 8 * quad) + j;
            w[j] = load4<T, MODE>(aw + int64_t(rank < p.r ? rank : 0) * p.h, h0 + permuted(col), p.h);
            if (rank >= p.r) w[j] = make_uint2(0, 0);
        }
        uint4 frag[4];
        transpose(w, frag);
#pragma unroll
        for (int e = 0; e < 4; ++e) as_bf16<T>(frag[e], fa[ks][e]);
    }
    f32x4 acc[RF][4];
#pragma unroll
    for (int f = 0; f < RF; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[f][e] = f32x4{0, 0, 0, 0};
    auto request = [&](int c, uint2 (&w)[8]) {
        int32_t tk[8];
        eight_tokens(tokens + c + 8 * quad, tk);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = row_load4<T, MODE>(p.x, row_offset<MODE>(tk[j], p.x_stride), col4, p.h);
    };
    auto step = [&](int c, const uint2 (&w)[8], uint2 (&next)[8]) {
        const uint4 *pu = packed + int64_t(c / 32) * (Packed<RP>::kColumns + Packed<RP>::kRows);
        BaseRow<T, MODE, BY_ROW> base[2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
            base[s].load(p.dx_base, p.dx_base == nullptr ? 0 : int64_t(tokens[c + 16 * s + col]) * p.dx_base_stride, out_col, p.h);
        uint4 rows[2][KS][HL];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int k = 0; k < HL; ++k) rows[s][ks][k] = has ? pu[Packed<RP>::kColumns + ((s * KS + ks) * HL + k) * kWave] : make_uint4(0, 0, 0, 0);
        request(c + 32 < tile.count ? c + 32 : c, next);
        if (has) {
            uint4 frag[4], part[4][NP];
            transpose(w, frag);
#pragma unroll
            for (int e = 0; e < 4; ++e) as_bf16<T>(frag[e], part[e]);
#pragma unroll
            for (int f = 0; f < RF; ++f) {
                uint4 v[3];
#pragma unroll
                for (int k = 0; k < 3; ++k) v[k] = pu[(f * 3 + k) * kWave];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[f][e] = outer<T>(part[e], v, acc[f][e]);
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f32x4 sum[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = f32x4{0, 0, 0, 0};
            if (has) {  // (A of another adapter was read in its place: 0 times its infinities would not be 0)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int k = 0; k < HL; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int q = 0; q < NP; ++q) sum[e] = mfma<Bf16>(fa[ks][e][q], rows[s][ks][k], sum[e]);
                if (any_odd(sum)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f32x4 kind = {0, 0, 0, 0};
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            const int ranks = RP <= 16 && quad >= 2 ? 0 : 8;  // (with R <= 16 the second half of the lanes holds low parts)
                            kind = mfma<Bf16>(first_entries(fa[ks][e][0], ranks),
                                              first_entries(pu[Packed<RP>::kColumns + (s * KS + ks) * HL * kWave], ranks), kind);
                        }
                        leading_kind(sum[e], kind);
                    }
                }
            }
            if (c + 16 * s + col < tile.count)
                base[s].store(static_cast<typename T::raw_t *>(p.dx) + int64_t(tokens[c + 16 * s + col]) * p.dx_stride, out_col, p.h, sum);
        }
    };
    uint2 even[8], odd[8];
    request(0, even);
    for (int c = 0; c < tile.count; c += 64) {
        step(c, even, odd);
        if (c + 32 >= tile.count) break;
        step(c + 32, odd, even);
    }
    if (!has) return;
#pragma unroll
    for (int f = 0; f < RF; ++f)
        if (any_odd(acc[f]))
            gradient_kind<T>(acc[f], tile.count, packed + f * 3 * kWave, Packed<RP>::kColumns + Packed<RP>::kRows, [&](int c, int j) {
                return row_load4<T, MODE>(p.x, row_offset<MODE>(tokens[c + 8 * quad + j], p.x_stride), col4, p.h);
            });
    float *da = tile.slot < 0 ? p.da + int64_t(tile.adapter) * p.r * p.h : p.da_part + int64_t(tile.slot) * p.r * p.h;
#pragma unroll
    for (int f = 0; f < RF; ++f) {
        const int rank = f * 16 + col;
        if (rank >= p.r) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = h0 + permuted(4 * quad + i);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (h + e < p.h) da[int64_t(rank) * p.h + h + e] = acc[f][e][i];
        }
    }
}

// grid (blocks of elements of dB, then of dA; adapters): adds the partial gradients of an adapter's further tiles in their
// order; zeros for an adapter without tokens.
struct FoldArgs {
    float *grad[2];
    const float *part[2];
    int64_t elements[2];
    int32_t blocks[2];
    LoraPlan plan;
};
__global__ __launch_bounds__(THREADS) void lora_fold_grads(FoldArgs p) {
    const int which = int(blockIdx.x) < p.blocks[0] ? 0 : 1, a = blockIdx.y;
    const int tiles = p.plan.list[which].per_adapter[2 * a], slot = p.plan.list[which].per_adapter[2 * a + 1];
    if (tiles == 1) return;
    const int64_t elements = p.elements[which], step = int64_t(p.blocks[which]) * THREADS;
    float *g = p.grad[which] + int64_t(a) * elements;
    for (int64_t i = int64_t(int(blockIdx.x) - (which ? p.blocks[0] : 0)) * THREADS + threadIdx.x; i < elements; i += step)
        g[i] = tiles == 0 ? 0.0f : add_parts(g[i], p.part[which] + int64_t(slot) * elements + i, tiles - 1, elements);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
inline size_t align_up(size_t n) { return (n + 255) / 256 * 256; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Shape { int64_t n, h, o, r, s; };

inline int check_shape(const char *what, int dtype, const Shape &d) {
    if (dtype != KA_DTYPE_BF16 && dtype != KA_DTYPE_F16) return fail(KA_ERR_BAD_ARG, "%s: dtype code %d is not bf16 or fp16", what, dtype);
    if (d.n < 0 || d.h < 1 || d.o < 1 || d.r < 1 || d.s < 1)
        return fail(KA_ERR_BAD_ARG, "%s: tokens %lld, widths %lld and %lld, rank %lld, adapters %lld must be positive", what,
                    (long long)d.n, (long long)d.h, (long long)d.o, (long long)d.r, (long long)d.s);
    if (d.r > MAX_RANK) return fail(KA_ERR_UNSUPPORTED, "%s: rank %lld > %d", what, (long long)d.r, MAX_RANK);
    if (d.s > MAX_ADAPTERS) return fail(KA_ERR_UNSUPPORTED, "%s: %lld adapters > %d", what, (long long)d.s, MAX_ADAPTERS);
    if (d.n > KA_LORA_MAX_TOKENS) return fail(KA_ERR_UNSUPPORTED, "%s: %lld tokens > %d", what, (long long)d.n, KA_LORA_MAX_TOKENS);
    if (d.h >= (int64_t(1) << 24) || d.o >= (int64_t(1) << 24)) return fail(KA_ERR_UNSUPPORTED, "%s: a width of 2^24 or more", what);
    return KA_OK;
}

inline int padded_rank(int64_t r) { return r <= 16 ? 16 : (r <= 32 ? 32 : (r <= 64 ? 64 : 128)); }

struct PlanLayout { size_t order, tiles[2], per_adapter[2], total; int64_t tokens[2], max_tiles[2]; };
inline PlanLayout plan_layout(int64_t n, int64_t s, int64_t tile0, int64_t tile1) {  // tile1 0: one list
    PlanLayout l{};
    const int64_t groups = s + 1 < n ? s + 1 : n;
    l.order = 256;  // behind the counts
    size_t at = l.order + align_up(size_t(n) * 4);
    for (int i = 0; i < 2; ++i) {
        l.tokens[i] = i == 0 ? tile0 : tile1;
        if (l.tokens[i] == 0) continue;
        l.max_tiles[i] = n / l.tokens[i] + groups;
        l.tiles[i] = at;
        l.per_adapter[i] = at + align_up(size_t(l.max_tiles[i]) * sizeof(LoraTile));
        at = l.per_adapter[i] + align_up(size_t(s) * 8);
    }
    l.total = at;
    return l;
}
inline LoraPlan plan_at(unsigned char *ws, const PlanLayout &l) {
    LoraPlan p{};
    p.order = reinterpret_cast<int32_t *>(ws + l.order);
    for (int i = 0; i < 2; ++i) {
        p.list[i].count = reinterpret_cast<int32_t *>(ws) + i;
        p.list[i].tiles = reinterpret_cast<LoraTile *>(ws + l.tiles[i]);
        p.list[i].per_adapter = reinterpret_cast<int32_t *>(ws + l.per_adapter[i]);
        p.list[i].tokens = int32_t(l.tokens[i]);
    }
    return p;
}

struct FwdLayout { PlanLayout plan; int64_t segments; bool split; size_t part, u, packed, total; };
inline FwdLayout fwd_layout(const Shape &d) {
    FwdLayout l;
    l.plan = plan_layout(d.n, d.s, FWD_TILE, 0);
    l.segments = ceil_div(d.h, SEG_STEPS * 32);
    // a workgroup per segment of H where the tiles alone are fewer than two per CU: 32 tokens, rank 64, H = O = 4096: 24 us a call,
    // 33 without; 8192 tokens, rank 16: 71 and 77
    l.split = l.segments > 1 && l.plan.max_tiles[0] < 512;
    l.part = l.plan.total;
    l.u = l.part + (l.split ? align_up(size_t(l.segments) * d.n * d.r * 4) : 0);
    l.packed = l.u + align_up(size_t(d.n) * d.r * 4);
    const int64_t rp = padded_rank(d.r);
    l.total = l.packed + size_t(l.plan.max_tiles[0]) * (rp == 16 ? RowFragments<16>::kTotal : rp == 32 ? RowFragments<32>::kTotal
                                                        : rp == 64 ? RowFragments<64>::kTotal : RowFragments<128>::kTotal) * sizeof(uint4);
    return l;
}

// The backward: outputs per wavefront (64 G) of the first pass, tokens per tile of both.
struct BwdLayout { PlanLayout plan; int64_t slots[2], blocks[2], folded; int groups; size_t packed, du_part, du_fold, db_part, da_part, total; };
// Tokens per tile such that `blocks` times the tiles make about `want` workgroups.
inline int64_t bwd_tile(int64_t n, int64_t blocks, int64_t want) {
    const int64_t tiles = ceil_div(want, blocks);
    int64_t tile = ceil_div(ceil_div(n, tiles), 32) * 32;
    return tile < 64 ? 64 : (tile > BWD_TILE_MAX ? BWD_TILE_MAX : tile);
}
inline BwdLayout bwd_layout(const Shape &d) {
    BwdLayout l;
    const int64_t small_blocks = ceil_div(d.o, 64 * WAVES);
    // 1024 outputs per workgroup instead of 256 where there are several rounds of workgroups all the same: fewer partial sums of
    // dy B, fewer wavefronts at a time.  us a call with 1024 and 256, rank 16: 1024 tokens x 128,256 outputs 145 / 135, 8192 x 14,336
    // 194 / 181, 2048 x 128,256 224 / 230, 8192 x 32,000 258 / 268, 4096 x 128,256 369 / 403.
    l.groups = padded_rank(d.r) == 16 && ceil_div(d.n, 64) * ceil_div(small_blocks, 4) >= 4000 ? 4 : 1;
    l.blocks[0] = ceil_div(d.o, 64 * WAVES * l.groups);
    l.blocks[1] = ceil_div(d.h, 64 * WAVES);
    // as many workgroups as the registers of the two kernels let reside at once
    const int64_t rp = padded_rank(d.r);
    const int64_t tile0 = bwd_tile(d.n, l.blocks[0], rp == 16 ? 1024 : (rp == 32 ? 512 : 256));
    const int64_t tile1 = bwd_tile(d.n, l.blocks[1], rp == 128 ? 256 : 512);
    l.slots[0] = d.n / tile0;
    l.slots[1] = d.n / tile1;
    l.plan = plan_layout(d.n, d.s, tile0, tile1);
    // fragments of u, then of dy B in the same place: 3 + 2 (or 4) KB per 32 tokens and 16 (or 32) ranks
    const size_t chunk = size_t(rp) / 16 * 3 * 1024 + (rp == 16 ? 2048 : size_t(rp) / 32 * 4 * 1024);
    l.packed = l.plan.total;
    l.du_part = l.packed + align_up(size_t(d.n / 32 + d.s + 1) * chunk);
    l.du_fold = l.du_part + align_up(size_t(l.blocks[0]) * d.n * d.r * 4);
    l.folded = l.blocks[0] > FOLD_PARTS ? ceil_div(l.blocks[0], FOLD_PARTS) : 0;
    l.db_part = l.du_fold + align_up(size_t(l.folded) * d.n * d.r * 4);
    l.da_part = l.db_part + align_up(size_t(l.slots[0]) * d.o * d.r * 4);
    l.total = l.da_part + align_up(size_t(l.slots[1]) * d.h * d.r * 4);
    return l;
}

inline bool aligned16(const void *p, int64_t stride) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0); }

// Calls launch(type, padded rank[, row mode]), each as a compile-time value.
template <typename F> void with_types(int dtype, int rp, F &&launch) {
    auto ranks = [&](auto type) {
        if (rp == 16) launch(type, std::integral_constant<int, 16>{});
        else if (rp == 32) launch(type, std::integral_constant<int, 32>{});
        else if (rp == 64) launch(type, std::integral_constant<int, 64>{});
        else launch(type, std::integral_constant<int, 128>{});
    };
    if (dtype == KA_DTYPE_BF16) ranks(Bf16{});
    else ranks(F16{});
}
template <typename F> void with_modes(int dtype, int rp, RowMode mode, F &&launch) {
    with_types(dtype, rp, [&](auto type, auto rank_c) {
        if (mode == ROWS_ALIGNED) launch(type, rank_c, std::integral_constant<int, ROWS_ALIGNED>{});
        else if (mode == ROWS_LOOSE) launch(type, rank_c, std::integral_constant<int, ROWS_LOOSE>{});
        else launch(type, rank_c, std::integral_constant<int, ROWS_SCALAR>{});
    });
}
inline RowMode row_mode(bool aligned, int64_t width) {
    return aligned && width % 8 == 0 ? ROWS_ALIGNED : (width >= 8 ? ROWS_LOOSE : ROWS_SCALAR);
}

}  // namespace
}  // namespace ka

KA_EXPORT size_t ka_lora_workspace_bytes(int64_t n_tokens, int64_t in_dim, int64_t out_dim, int64_t rank, int64_t n_adapters,
                                         int backward) {
    const ka::Shape d{n_tokens, in_dim, out_dim, rank, n_adapters};
    if (ka::check_shape("lora", KA_DTYPE_BF16, d) != KA_OK || n_tokens == 0) return 0;
    return backward ? ka::bwd_layout(d).total : ka::fwd_layout(d).total;
}

KA_EXPORT int ka_lora_linear(int dtype, const void *base, int64_t base_stride, const void *hidden, int64_t hidden_stride,
                             const void *lora_a, const void *lora_b, const int64_t *adapter_ids, const float *scaling,
                             float scale, void *out, int64_t out_stride, float *out_shrunk, int64_t n_tokens, int64_t in_dim,
                             int64_t out_dim, int64_t rank, int64_t n_adapters, void *workspace, size_t workspace_bytes,
                             void *hip_stream) {
    using namespace ka;
    const Shape d{n_tokens, in_dim, out_dim, rank, n_adapters};
    int rc = check_shape("lora", dtype, d);
    if (rc != KA_OK) return rc;
    if (n_tokens == 0) return KA_OK;
    if (hidden == nullptr || lora_a == nullptr || adapter_ids == nullptr || (out != nullptr && (base == nullptr || lora_b == nullptr)) ||
        (out == nullptr && out_shrunk == nullptr))
        return fail(KA_ERR_BAD_ARG, "lora: null base / hidden / lora_a / lora_b / adapter_ids / out pointer");
    if ((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(lora_a) |
         reinterpret_cast<uintptr_t>(lora_b) | reinterpret_cast<uintptr_t>(out)) % 2 != 0)
        return fail(KA_ERR_BAD_ARG, "lora: a matrix is not aligned to its elements");
    if ((out != nullptr && (base_stride < out_dim || out_stride < out_dim)) || hidden_stride < in_dim)
        return fail(KA_ERR_BAD_ARG, "lora: a row stride is smaller than its row");
    const FwdLayout l = fwd_layout(d);
    if (workspace == nullptr || workspace_bytes < l.total)
        return fail(KA_ERR_WORKSPACE, "lora: workspace of %zu B, need %zu B", workspace == nullptr ? size_t(0) : workspace_bytes, l.total);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(KA_ERR_BAD_ARG, "lora: workspace is not 16-byte aligned");
    const RowMode shrink_mode = row_mode(aligned16(hidden, hidden_stride) && aligned16(lora_a, 0), in_dim);
    const RowMode expand_mode = row_mode(aligned16(base, base_stride) && aligned16(out, out_stride) && aligned16(lora_b, 0) && rank % 8 == 0, out_dim);
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    const LoraPlan plan = plan_at(ws, l.plan);
    // Few tokens: one workgroup per token and segment, which needs no plan, and the plan made by one more beside them; every token
    // reads its A from L2.  H = O = 4096, us a call with and without: 1 token, rank 16: 23 / 29; 512, rank 16: 26 / 30;
    // 1024, rank 16: 41 / 28; 128, rank 64: 25 / 31; 512, rank 32: 35 / 29.
    const bool one = n_tokens * rank <= 8192 && n_tokens <= 512;
    if (!one) {
        hipLaunchKernelGGL(lora_plan, dim3(1), dim3(PLAN_THREADS), 0, stream, adapter_ids, int(n_tokens), int(n_adapters), 1, plan);
        rc = check_hip(hipGetLastError(), "lora launch (plan)");
        if (rc != KA_OK) return rc;
    }
    // u whole, or its segments for lora_expand to add
    float *u = out_shrunk != nullptr ? out_shrunk : reinterpret_cast<float *>(ws + l.u);
    float *parts = reinterpret_cast<float *>(ws + l.part);
    ShrinkArgs sa{};
    sa.x = hidden;
    sa.a = lora_a;
    sa.x_stride = hidden_stride;
    sa.ids = adapter_ids;
    sa.scaling = scaling;
    sa.scale = scale;
    sa.n = int32_t(n_tokens);
    sa.h = int32_t(in_dim);
    sa.r = int32_t(rank);
    sa.s = int32_t(n_adapters);
    sa.segments = int32_t(l.segments);
    sa.split = l.split ? 1 : 0;
    sa.out = l.split ? parts : u;
    sa.plan = plan;
    const int rp = padded_rank(rank);
    const dim3 shrink_grid{unsigned(l.split ? l.segments : 1), unsigned(one ? n_tokens + 1 : l.plan.max_tiles[0])};
    with_modes(dtype, rp, shrink_mode, [&](auto type, auto rank_c, auto mode_c) {
        using T = decltype(type);
        constexpr int RP = decltype(rank_c)::value, MODE = decltype(mode_c)::value;
        if (one) hipLaunchKernelGGL((lora_shrink<T, RP, MODE, true>), shrink_grid, dim3(THREADS), 0, stream, sa);
        else hipLaunchKernelGGL((lora_shrink<T, RP, MODE, false>), shrink_grid, dim3(THREADS), 0, stream, sa);
    });
    rc = check_hip(hipGetLastError(), "lora launch (shrink)");
    if (rc != KA_OK) return rc;
    // (a call of few tokens saves a launch: its segments are added by the few workgroups that read them)
    const bool parted = l.split && one && out != nullptr;
    if (l.split && out == nullptr) {
        hipLaunchKernelGGL(lora_fold_rows, dim3(unsigned(ceil_div(n_tokens * rank, THREADS))), dim3(THREADS), 0, stream,
                           parts, int(l.segments), n_tokens, int(rank), adapter_ids, int(n_adapters), scaling, scale, u);
        rc = check_hip(hipGetLastError(), "lora launch (fold)");
        if (rc != KA_OK) return rc;
    }
    uint4 *packed = reinterpret_cast<uint4 *>(ws + l.packed);
    if (out != nullptr && !parted) {
        PackRowsArgs pa{};
        pa.part = l.split ? parts : u;
        pa.out_shrunk = l.split ? out_shrunk : nullptr;
        pa.scaling = scaling;
        pa.scale = scale;
        pa.parts = l.split ? int32_t(l.segments) : 1;
        pa.scaled = l.split ? 1 : 0;
        pa.r = int32_t(rank);
        pa.n = n_tokens;
        pa.out = packed;
        pa.plan = plan;
        with_types(dtype, rp, [&](auto, auto rank_c) {
            constexpr int RP = decltype(rank_c)::value;
            hipLaunchKernelGGL((lora_pack_rows<RP>), dim3(unsigned(l.plan.max_tiles[0])), dim3(THREADS), 0, stream, pa);
        });
        rc = check_hip(hipGetLastError(), "lora launch (pack)");
        if (rc != KA_OK) return rc;
    }
    if (out == nullptr) return KA_OK;
    ExpandArgs ea{};
    ea.base = base;
    ea.b = lora_b;
    ea.out = out;
    ea.base_stride = base_stride;
    ea.out_stride = out_stride;
    ea.packed = packed;
    ea.u = parts;
    ea.out_shrunk = out_shrunk;
    ea.scaling = scaling;
    ea.scale = scale;
    ea.n = n_tokens;
    ea.parts = int32_t(l.segments);
    ea.o = int32_t(out_dim);
    ea.r = int32_t(rank);
    ea.in_place = out == base && out_stride == base_stride ? 1 : 0;
    ea.plan = plan;
    // groups of 64 outputs per wavefront: as many as leave about 1024 workgroups
    const int64_t blocks1 = ceil_div(out_dim, 64 * WAVES);
    int64_t groups = blocks1 * l.plan.max_tiles[0] / 1024;
    groups = groups < 1 ? 1 : (groups > 8 ? 8 : groups);
    ea.groups = int32_t(groups);
    const dim3 expand_grid{unsigned(ceil_div(out_dim, 64 * WAVES * groups)), unsigned(l.plan.max_tiles[0])};
    with_modes(dtype, rp, expand_mode, [&](auto type, auto rank_c, auto mode_c) {
        using T = decltype(type);
        constexpr int RP = decltype(rank_c)::value, MODE = decltype(mode_c)::value;
        if (parted) hipLaunchKernelGGL((lora_expand<T, RP, MODE, true>), expand_grid, dim3(THREADS), 0, stream, ea);
        else hipLaunchKernelGGL((lora_expand<T, RP, MODE, false>), expand_grid, dim3(THREADS), 0, stream, ea);
    });
    return check_hip(hipGetLastError(), "lora launch (expand)");
}

KA_EXPORT int ka_lora_linear_backward(int dtype, const void *grad_out, int64_t grad_stride, const void *hidden,
                                      int64_t hidden_stride, const void *lora_a, const void *lora_b, const int64_t *adapter_ids,
                                      const float *scaling, float scale, const float *shrunk, const void *dhidden_base,
                                      int64_t dhidden_base_stride, void *dhidden, int64_t dhidden_stride, float *dlora_a,
                                      float *dlora_b, int64_t n_tokens, int64_t in_dim, int64_t out_dim, int64_t rank,
                                      int64_t n_adapters, void *workspace, size_t workspace_bytes, void *hip_stream) {
    using namespace ka;
    const Shape d{n_tokens, in_dim, out_dim, rank, n_adapters};
    int rc = check_shape("lora backward", dtype, d);
    if (rc != KA_OK) return rc;
    if (n_tokens == 0) return fail(KA_ERR_BAD_ARG, "lora backward: no tokens (the gradients would be zero)");
    if (grad_out == nullptr || hidden == nullptr || lora_a == nullptr || lora_b == nullptr || adapter_ids == nullptr ||
        shrunk == nullptr || dhidden == nullptr || dlora_a == nullptr || dlora_b == nullptr)
        return fail(KA_ERR_BAD_ARG, "lora backward: null grad_out / hidden / lora_a / lora_b / adapter_ids / shrunk / result pointer");
    if ((reinterpret_cast<uintptr_t>(grad_out) | reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(lora_a) |
         reinterpret_cast<uintptr_t>(lora_b) | reinterpret_cast<uintptr_t>(dhidden_base) | reinterpret_cast<uintptr_t>(dhidden)) % 2 != 0)
        return fail(KA_ERR_BAD_ARG, "lora backward: a matrix is not aligned to its elements");
    if (grad_stride < out_dim || hidden_stride < in_dim || dhidden_stride < in_dim || (dhidden_base != nullptr && dhidden_base_stride < in_dim))
        return fail(KA_ERR_BAD_ARG, "lora backward: a row stride is smaller than its row");
    const BwdLayout l = bwd_layout(d);
    if (workspace == nullptr || workspace_bytes < l.total)
        return fail(KA_ERR_WORKSPACE, "lora backward: workspace of %zu B, need %zu B", workspace == nullptr ? size_t(0) : workspace_bytes, l.total);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(KA_ERR_BAD_ARG, "lora backward: workspace is not 16-byte aligned");
    constexpr int64_t NARROW = int64_t(1) << 32;  // bytes of a matrix that offsets of 32 bits reach
    const RowMode out_mode = row_mode(aligned16(grad_out, grad_stride) && n_tokens * grad_stride * 2 < NARROW, out_dim);
    const RowMode in_mode = row_mode(aligned16(hidden, hidden_stride) && aligned16(dhidden_base, dhidden_base_stride) &&
                                     aligned16(dhidden, dhidden_stride) && aligned16(lora_a, 0) && n_tokens * hidden_stride * 2 < NARROW, in_dim);
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    const LoraPlan plan = plan_at(ws, l.plan);
    hipLaunchKernelGGL(lora_plan, dim3(1), dim3(PLAN_THREADS), 0, stream, adapter_ids, int(n_tokens), int(n_adapters), 2, plan);
    rc = check_hip(hipGetLastError(), "lora backward launch (plan)");
    if (rc != KA_OK) return rc;
    const int rp = padded_rank(rank);
    uint4 *packed = reinterpret_cast<uint4 *>(ws + l.packed);
    float *du_part = reinterpret_cast<float *>(ws + l.du_part);
    float *db_part = reinterpret_cast<float *>(ws + l.db_part), *da_part = reinterpret_cast<float *>(ws + l.da_part);
    auto pack = [&](const float *part, int64_t parts, bool scaled) {
        PackArgs pa{};
        pa.part = part;
        pa.parts = int32_t(parts);
        pa.r = int32_t(rank);
        pa.rows = scaled ? 1 : 0;
        pa.n = n_tokens;
        pa.scaling = scaling;
        pa.scale = scale;
        pa.scaled = scaled ? 1 : 0;
        pa.out = packed;
        pa.plan = plan;
        const dim3 grid{unsigned(l.plan.tokens[0] / 32), unsigned(l.plan.max_tiles[0])};
        with_types(dtype, rp, [&](auto, auto rank_c) {
            constexpr int RP = decltype(rank_c)::value;
            hipLaunchKernelGGL((lora_pack<RP>), grid, dim3(THREADS), 0, stream, pa);
        });
        return check_hip(hipGetLastError(), "lora backward launch (pack)");
    };
    rc = pack(shrunk, 1, false);
    if (rc != KA_OK) return rc;
    BwdOutArgs oa{};
    oa.dy = grad_out;
    oa.b = lora_b;
    oa.dy_stride = grad_stride;
    oa.u = packed;
    oa.n = int32_t(n_tokens);
    oa.o = int32_t(out_dim);
    oa.r = int32_t(rank);
    oa.db = dlora_b;
    oa.db_part = db_part;
    oa.du_part = du_part;
    oa.plan = plan;
    const dim3 out_grid{unsigned(l.blocks[0]), unsigned(l.plan.max_tiles[0])};
    with_modes(dtype, rp, out_mode, [&](auto type, auto rank_c, auto mode_c) {
        using T = decltype(type);
        constexpr int RP = decltype(rank_c)::value, MODE = decltype(mode_c)::value;
        if constexpr (RP == 16) {
            if (l.groups == 4) {
                hipLaunchKernelGGL((lora_bwd_out<T, RP, 4, MODE>), out_grid, dim3(THREADS), 0, stream, oa);
                return;
            }
        }
        hipLaunchKernelGGL((lora_bwd_out<T, RP, 1, MODE>), out_grid, dim3(THREADS), 0, stream, oa);
    });
    rc = check_hip(hipGetLastError(), "lora backward launch (out)");
    if (rc != KA_OK) return rc;
    float *du_fold = reinterpret_cast<float *>(ws + l.du_fold);
    if (l.folded > 0) {
        hipLaunchKernelGGL(lora_fold_parts, dim3(unsigned(ceil_div(n_tokens * rank, THREADS)), unsigned(l.folded)), dim3(THREADS), 0, stream,
                           du_part, int(l.blocks[0]), n_tokens * rank, du_fold);
        rc = check_hip(hipGetLastError(), "lora backward launch (fold)");
        if (rc != KA_OK) return rc;
    }
    rc = l.folded > 0 ? pack(du_fold, l.folded, true) : pack(du_part, l.blocks[0], true);
    if (rc != KA_OK) return rc;
    BwdInArgs ia{};
    ia.x = hidden;
    ia.a = lora_a;
    ia.dx_base = dhidden_base;
    ia.dx = dhidden;
    ia.x_stride = hidden_stride;
    ia.dx_base_stride = dhidden_base_stride;
    ia.dx_stride = dhidden_stride;
    ia.du = packed;
    ia.h = int32_t(in_dim);
    ia.r = int32_t(rank);
    ia.da = dlora_a;
    ia.da_part = da_part;
    ia.plan = plan;
    const dim3 in_grid{unsigned(l.blocks[1]), unsigned(l.plan.max_tiles[1])};
    with_modes(dtype, rp, in_mode, [&](auto type, auto rank_c, auto mode_c) {
        using T = decltype(type);
        constexpr int RP = decltype(rank_c)::value, MODE = decltype(mode_c)::value;
        hipLaunchKernelGGL((lora_bwd_in<T, RP, MODE>), in_grid, dim3(THREADS), 0, stream, ia);
    });
    rc = check_hip(hipGetLastError(), "lora backward launch (in)");
    if (rc != KA_OK) return rc;
    FoldArgs fa{};
    fa.plan = plan;
    fa.grad[0] = dlora_b;
    fa.grad[1] = dlora_a;
    fa.part[0] = db_part;
    fa.part[1] = da_part;
    for (int i = 0; i < 2; ++i) {
        fa.elements[i] = (i == 0 ? out_dim : in_dim) * rank;
        const int64_t blocks = ceil_div(fa.elements[i], THREADS);
        fa.blocks[i] = int32_t(blocks < 2048 ? blocks : 2048);
    }
    hipLaunchKernelGGL(lora_fold_grads, dim3(unsigned(fa.blocks[0] + fa.blocks[1]), unsigned(n_adapters)), dim3(THREADS), 0, stream, fa);
    return check_hip(hipGetLastError(), "lora backward launch (gradients)");
}
