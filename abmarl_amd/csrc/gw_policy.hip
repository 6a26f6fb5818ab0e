// gw_policy.hip — drawing actions from a policy's logits, and the clipped
// policy loss with its gradient (include/gw_learn.h gw_policy_*).
//
// A row of logits is a few softmaxes side by side (its heads), p = e^(z - top) / S:
//   log p(action) = sum of (x - log S) at the heads' choices, x = z - top
//   H  = sum over heads of log S - T / S,          T = sum of e^x x
//   KL = sum over heads of U / Sr + log(S / Sr),   U = sum of e^y (y - x), y = ref's x
// so S, T, Sr, U of one walk over a row give the loss, and they and the exponentials
// give its gradient.  Drawing takes the largest z + noise of a head (the lowest
// choice of equals).  A row is read once and written once (the gradient); there
// are three layouts: rows of up to 48 choices a lane each, one wide head a group of
// lanes, and everything else a workgroup a row.
#include <stdarg.h>
#include <stdio.h>

#include <type_traits>

#include "gw_learn.hpp"

static thread_local char g_err[512];

void gw_learn_set_err(const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
}

namespace {

// the heads, by value in the launch's arguments: no device table to keep
struct Heads {
    int32_t n, act_dim, width;                  // heads, columns of an action row, choices
    int32_t off[GW_MAX_HEADS + 1];
    int32_t low[GW_MAX_HEADS];
    int16_t slot[GW_MAX_HEADS];
    int16_t large[GW_MAX_HEADS], n_large;       // the heads of more than LANE_HEAD choices
};
constexpr int LANE_HEAD = 16;

struct SampleArgs {
    const void* logits; int64_t ld, rows;
    const float* noise;
    const uint8_t* mask; int64_t mask_rows;
    int32_t* actions; float* logp; float* entropy;
};

struct LossArgs {
    const void* logits; const void* ref; int64_t ld, ld_ref, rows;
    const int32_t* actions; const float* advantage; const float* old_logp;
    const uint8_t* valid; const uint8_t* mask; int64_t mask_rows;
    float lo, hi, kl, entropy;                  // 1 - clip_low, 1 + clip_high, coefficients
    float denominator; const float* denominator_at;
    float scale; const float* upstream;
    float* out; float* stats; float* logp; void* grad;      // out: the loss
    const int32_t* counts; int32_t n_counts;    // valid rows per block of count_kernel
    double* partial;                            // [blocks][N_SUMS]
};

enum { S_PG, S_KL, S_H, S_CLIP, S_COUNT, N_SUMS };

// ------------------------------------------------------------ group of G threads
template <int G>
struct Group {
    float* box;                                 // G / 64 floats of LDS
    __device__ __forceinline__ float max(float v)
    {
        v = wave_max_nan(v);
        if constexpr (G > WAVE) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
            __syncthreads();
            v = box[0];
#pragma unroll
            for (int w = 1; w < G / WAVE; w++) v = max_nan(v, box[w]);
        }
        return v;
    }
    __device__ __forceinline__ float sum(float v)
    {
        v = wave_sum(v);
        if constexpr (G > WAVE) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
            __syncthreads();
            v = box[0];
#pragma unroll
            for (int w = 1; w < G / WAVE; w++) v += box[w];
        }
        return v;
    }
};

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// The largest |top| for which logits become exponents by one fma, z log2(e) -
// round(top log2(e)).  The rounding shifts all exponents of a row alike, which cancels in
// what they are used for, as long as all of them are made this way; here it is under 2^-7.
// (At 1e10 it would be 440, and 2^440 infinite.)  Every float16 is in.
constexpr float NEAR_TOP = 65536.f;
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// 1/x and the logarithm of sums of exponentials and of their quotients: the
// hardware's, and a step of Newton's behind it.  The hardware's logarithm cuts off:
// over 2^20 values from 2^-10 to 2^3 its mean error was -1.6e-7 (at most 9.5e-7), and
// a log-probability of eleven heads was 8e-7 too high in the mean.
// log x = l + (x e^-l - 1) takes that to 4e-8, as 2^x errs by 2.6e-8 (root mean square;
// mean -3e-9); 1/x by 2.8e-8 (mean -6e-9, which a KL of eleven heads shows).  Twice a
// head, it costs the narrow rows 2 to 3% (5.2 M rows of 3, 3, 2: 143 to 147 us).
__device__ __forceinline__ float rcp_of(float x)
{
    const float r = __builtin_amdgcn_rcpf(x);
    return fmaf(fmaf(-x, r, 1.f), r, r);
}
__device__ __forceinline__ float log_of(float x)
{
    const float l = __builtin_amdgcn_logf(x);
    return fmaf(l, LN2, fmaf(x, exp2_of(-l), -1.f));
}

// v - m of finite logits may pass the largest number; where its exponential is 0, so
// must be their product.  NaN stays.
__device__ __forceinline__ float below(float v, float m)
{
    const float x = v - m;
    return x < -1e30f ? -1e30f : x;
}

template <class T>
__device__ __forceinline__ float logit_at(const T* row, const uint8_t* mask, int j)
{
    return (mask && !mask[j]) ? NEG_INF : (float)row[j];
}

// Rows that neither fit a thread nor are one head: a row by a workgroup of G
// threads.  Heads of up to LANE_HEAD choices are walked by one lane each (the
// cells of an attack window are dozens of heads of a few choices), larger ones
// by the whole group, their choices strided over it.  Right for every layout.
// G grows with the row, so that a large head's walk stays short.  Where a wave
// takes a row (below STAGED_ROW choices) the row is copied to LDS first, and the
// gradient leaves from there: the walks over heads would read the memory in pieces of
// a head, one after the other.  65536 rows of 51 heads (214 choices bf16): drawn in
// 77 us (171 without), loss and gradient with ref 174 us (358), where the bytes take
// 19 us in either; the heads' walks, a few choices each, one after another, bound it.
constexpr int STAGED_ROW = 1024;

// a row to LDS as float, its loads side by side and four in flight; masked choices as -inf
template <class T, int G>
__device__ __forceinline__ void stage_row(const T* row, const uint8_t* mask, int width, float* to)
{
    for (int j = threadIdx.x; j < width; j += 4 * G) {
        T v[4];
        uint8_t m[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int at = j + k * G < width ? j + k * G : width - 1;
            v[k] = row[at];
            m[k] = mask ? mask[at] : 1;
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (j + k * G < width) to[j + k * G] = m[k] ? (float)v[k] : NEG_INF;
    }
}

// A lane's first head, read once: what stands at a lane's own place in the
// arguments is a load from memory.
struct OwnHead {
    int lo, hi, slot, low;
    __device__ __forceinline__ OwnHead(const Heads& h, int d) : lo(h.off[d]), hi(h.off[d + 1]), slot(h.slot[d]), low(h.low[d]) {}
};

template <class T, int G>
__global__ __launch_bounds__(G) void sample_rows_kernel(SampleArgs a, Heads h)
{
    __shared__ float box[G / WAVE];
    __shared__ float best_s[G / WAVE];
    __shared__ int best_i[G / WAVE];
    extern __shared__ float lds_row[];          // STAGED: the row, its noise
    constexpr bool STAGED = G == WAVE;
    Group<G> grp{box};
    const int tid = threadIdx.x;
    const OwnHead own(h, tid < h.n ? tid : 0);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* z = (const T*)a.logits + row * a.ld;
        const float* noise = a.noise ? a.noise + row * h.width : nullptr;
        const uint8_t* mask = a.mask ? a.mask + (row % a.mask_rows) * h.width : nullptr;
        int32_t* act = a.actions + row * h.act_dim;
        if constexpr (STAGED) {
            stage_row<T, G>(z, mask, h.width, lds_row);
            if (noise) stage_row<float, G>(noise, nullptr, h.width, lds_row + h.width);
            __syncthreads();
        }
        const auto logit = [&](int j) __attribute__((always_inline)) { return STAGED ? lds_row[j] : logit_at(z, mask, j); };
        const auto score = [&](int j, float v) __attribute__((always_inline)) {
            return noise ? v + (STAGED ? lds_row[h.width + j] : noise[j]) : v;
        };
        if (h.n < h.act_dim)
            for (int c = tid; c < h.act_dim; c += G) {
                bool owned = false;
                for (int d = 0; d < h.n; d++) owned |= h.slot[d] == c;
                if (!owned) act[c] = 0;
            }
        float logp = 0.f, entropy = 0.f;                 // of this lane's heads; the group's in lane 0
        for (int d = tid; d < h.n; d += G) {
            const OwnHead mine = d == tid ? own : OwnHead(h, d);
            const int lo = mine.lo, hi = mine.hi;
            if (hi - lo > LANE_HEAD) continue;
            float m = NEG_INF, bs = NEG_INF, at = 0.f, s = 0.f, t = 0.f;
            int bi = -1;
            for (int j = lo; j < hi; j++) {
                const float v = logit(j);
                if (v == NEG_INF) continue;
                m = max_nan(m, v);
                const float sc = score(j, v);
                if (sc > bs || (bi < 0 && sc == bs)) { bs = sc; bi = j; at = v; }
            }
            if (m != NEG_INF) {
                for (int j = lo; j < hi; j++) {
                    const float v = logit(j);
                    if (v == NEG_INF) continue;
                    const float x = below(v, m), e = expf(x);
                    s += e;
                    t += e * x;
                }
                const float log_s = log_of(s);
                logp += (at - m) - log_s;
                entropy += log_s - t / s;
            }
            act[mine.slot] = mine.low + (bi < 0 ? 0 : bi - lo);
        }
        double row_logp = 0.;
        float row_entropy = 0.f;
        for (int i = 0; i < h.n_large; i++) {
            const int d = h.large[i], lo = h.off[d], hi = h.off[d + 1];
            float m = NEG_INF, bs = NEG_INF;
            int bi = INT32_MAX;
            for (int j = lo + tid; j < hi; j += G) {
                const float v = logit(j);
                if (v == NEG_INF) continue;
                m = max_nan(m, v);
                const float s = score(j, v);
                if (s > bs || (s == bs && j < bi)) { bs = s; bi = j; }
            }
            m = grp.max(m);
            if (m == NEG_INF) {                          // no choice in this head
                if (tid == 0) act[h.slot[d]] = h.low[d];
                continue;
            }
#pragma unroll
            for (int o = WAVE / 2; o > 0; o >>= 1) {
                const float os = __shfl_xor(bs, o);
                const int oi = __shfl_xor(bi, o);
                if (os > bs || (os == bs && oi < bi)) { bs = os; bi = oi; }
            }
            if constexpr (G > WAVE) {
                __syncthreads();
                if ((tid & 63) == 0) { best_s[tid >> 6] = bs; best_i[tid >> 6] = bi; }
                __syncthreads();
                for (int w = 0; w < G / WAVE; w++)
                    if (best_s[w] > bs || (best_s[w] == bs && best_i[w] < bi)) { bs = best_s[w]; bi = best_i[w]; }
            }
            if (bi == INT32_MAX) bi = lo;                // every score NaN
            float s = 0.f, t = 0.f;
            for (int j = lo + tid; j < hi; j += G) {
                const float v = logit(j);
                if (v == NEG_INF) continue;
                const float x = below(v, m), e = expf(x);
                s += e;
                t += e * x;
            }
            s = grp.sum(s);
            t = grp.sum(t);
            const float log_s = log_of(s);
            row_logp += (double)(logit(bi) - m) - (double)log_s;
            row_entropy += log_s - t / s;
            if (tid == 0) act[h.slot[d]] = h.low[d] + (bi - lo);
        }
        logp = grp.sum(logp);
        entropy = grp.sum(entropy);
        if (tid == 0) {
            if (a.logp) a.logp[row] = (float)(row_logp + (double)logp);
            if (a.entropy) a.entropy[row] = row_entropy + entropy;
        }
        if constexpr (STAGED) __syncthreads();           // the next row goes where this one is
    }
}

// what a row's loss needs besides its heads' softmax
struct RowLoss {
    float logp, pull, pg, kl, entropy;          // pull: d(-surrogate)/dL = -ratio A where not clipped
    bool clipped;
};

// (L is a sum of numbers near its own size: in double its difference to
// old_logp, which is near 0, is exact to the heads' own errors)
__device__ __forceinline__ RowLoss row_loss(const LossArgs& a, float adv, float old, double logp, bool possible, float kl, float entropy)
{
    RowLoss r;
    r.logp = possible ? (float)logp : NEG_INF;
    const float ratio = possible ? expf((float)(logp - (double)old)) : 0.f;
    const float clamped = fminf(fmaxf(ratio, a.lo), a.hi);
    // (a ratio past the largest number is no NaN beside an advantage of 0)
    const float free = ratio == -NEG_INF && adv == 0.f ? 0.f : ratio * adv, held = (ratio != ratio ? ratio : clamped) * adv;
    r.clipped = held < free;
    r.pull = r.clipped ? 0.f : -free;
    r.pg = r.clipped ? -held : -free;
    r.kl = kl;
    r.entropy = entropy;
    return r;
}

// M as it is given, or -1: the valid rows are to be counted
__device__ __forceinline__ float given_rows(const LossArgs& a)
{
    return a.denominator > 0.f ? a.denominator : a.denominator_at ? fmaxf(*a.denominator_at, 0.f) : -1.f;
}

// 1/M, or 0 where there is nothing to take a mean of
__device__ __forceinline__ float inverse_rows(const LossArgs& a)
{
    float m = given_rows(a);
    if (m < 0.f) {
        m = (float)a.rows;
        if (a.counts) {
            // (every wave adds the blocks' counts)
            int64_t n = 0;
            for (int i = threadIdx.x & 63; i < a.n_counts; i += WAVE) n += a.counts[i];
            m = (float)wave_sum(n);
        }
    }
    return m > 0.f ? 1.f / m : 0.f;
}

// the blocks' sums to gw_policy_loss's loss and stats
__device__ __forceinline__ void write_out(const LossArgs& a, const double* s)
{
    const float given = given_rows(a);
    const double m = given >= 0.f ? (double)given : s[S_COUNT];
    const double inv = m > 0. ? 1. / m : 0.;
    a.out[0] = (float)((s[S_PG] + (double)a.kl * s[S_KL] - (double)a.entropy * s[S_H]) * inv);
    a.stats[0] = (float)(s[S_PG] * inv);
    a.stats[1] = (float)(s[S_KL] * inv);
    a.stats[2] = (float)(s[S_H] * inv);
    a.stats[3] = (float)(s[S_CLIP] * inv);
    a.stats[4] = (float)m;
}

// ------------------------------------------------------------ rows out of registers
template <class T, int CM>
__device__ __forceinline__ void store_row(T* row, int width, const float* v)
{
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < CM / PER; u++) {
        if (u * PER >= width) continue;
        T t[PER];
#pragma unroll
        for (int e = 0; e < PER; e++) t[e] = (T)v[u * PER + e];
        uint4 w;
        __builtin_memcpy(&w, t, 16);
        ((uint4*)row)[u] = w;
    }
}

// a lane's row into the wave's tile in LDS (rows side by side)
template <class T, int CM>
__device__ __forceinline__ void write_tile(T* row, int width, const float* v)
{
    if (sizeof(T) == 2 && (width & 1) == 0) {
#pragma unroll
        for (int j = 0; j < CM; j += 2) {
            if (j >= width) continue;
            const T t[2] = {(T)v[j], (T)v[j + 1]};
            uint32_t w;
            __builtin_memcpy(&w, t, sizeof(T) == 2 ? 4 : 0);
            ((uint32_t*)row)[j / 2] = w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < CM; j++)
            if (j < width) row[j] = (T)v[j];
    }
}

// the tile to memory, side by side there too
template <class T>
__device__ __forceinline__ void copy_tile(const T* tile, T* to, int n, bool wide, int lane)
{
    constexpr int PER = 16 / sizeof(T);
    int done = 0;
    if (wide) {
        done = n / PER * PER;
        for (int i = lane; i < n / PER; i += WAVE) ((uint4*)to)[i] = ((const uint4*)tile)[i];
    }
    for (int i = done + lane; i < n; i += WAVE) to[i] = tile[i];
}

// a workgroup's sums: to its place among the partial ones, or, where it is the only one, to out
template <int WAVES>
__device__ __forceinline__ void block_sums(const LossArgs& a, double* s)
{
    __shared__ double box[WAVES][N_SUMS];
#pragma unroll
    for (int k = 0; k < N_SUMS; k++) s[k] = wave_sum(s[k]);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0)
            for (int k = 0; k < N_SUMS; k++) box[threadIdx.x >> 6][k] = s[k];
        __syncthreads();
        if (threadIdx.x != 0) return;
        for (int w = 1; w < WAVES; w++)
            for (int k = 0; k < N_SUMS; k++) s[k] += box[w][k];
    }
    if (threadIdx.x != 0) return;
    if (gridDim.x == 1) write_out(a, s);
    else
        for (int k = 0; k < N_SUMS; k++) a.partial[(int64_t)k * gridDim.x + blockIdx.x] = s[k];
}

// ------------------------------------------------------------- narrow rows
// A thread a row, the whole row in registers (CM: the width, rounded up).
// Where the heads begin and end is uniform, so the sweeps over a row are
// unrolled and a head's end is a scalar branch: no lane of a wave idles, no
// reduction crosses lanes, and the memory sees each value once.  A choice that
// does not exist holds NO_CHOICE, whose exponential is 0.
//
// Large calls are bound by the vector units and by waits between a tile's loads
// and its sums, with the registers a row takes for a limit on waves:
//   5.2 M rows of 3, 3, 2 bf16, ref and valid flags, loss and gradient: 147 us,
//     382 MB at 2.6 TB/s (a copy: 5.2); 87 lane instructions a choice, about 93 us of issue;
//   1.0 M rows of 28 choices f16, masks of 256 lanes: loss 65 us, gradient 95 us;
//   262144 rows of 3, 3, 2 bf16 drawn with their noise: 8.2 us, 17.6 MB (3.4 us).
// Forcing more waves a CU by launch bounds spilt registers and was slower.
// CM goes in steps of 8 above 16, as what lies behind the width is worked on too:
// 500000 rows of 9, 9, 3 bf16 with ref, loss and gradient: 52 us by 24, 84 us by 32;
// of 15, 15, 5: 114 us by 40, 126 us by 48.
constexpr int NARROW = 48;
constexpr float NO_CHOICE = -3.2e38f;           // (nobody masks by this number)

struct Small {
    int32_t n, act_dim, width, owned;           // owned: every action column has a head
    uint64_t starts, ends;                      // bit j: choice j is a head's first, last
    int32_t low[NARROW + 3];                    // (read in fours)
    int16_t slot[NARROW + 3];
    uint8_t first[NARROW + 3], size[NARROW + 3];  // a head's first choice, how many
    int32_t unit, unit_ref, unit_mask, unit_grad, unit_noise;  // bytes that a row's loads and stores may take at once
};

// A wave's 64 rows: a uniform first one and the lane's own behind it (the last
// row again for lanes behind it)
struct Tile {
    int64_t base;
    uint32_t l;
    bool there;
    __device__ __forceinline__ Tile(int64_t tile, int64_t rows, int lane) : base(tile * WAVE)
    {
        const int64_t left = rows - 1 - base;
        there = lane <= left;
        l = there ? (uint32_t)lane : (uint32_t)left;
    }
};

// The heads' ends are tested dozens of times a row.  Without this the
// compiler keeps every test's outcome over all rows, in more scalar
// registers than there are.
struct Bounds {
    uint64_t starts, ends;
    int32_t width, n, unit, unit_ref;
    __device__ __forceinline__ explicit Bounds(const Small& h)
        : starts(h.starts), ends(h.ends), width(h.width), n(h.n), unit(h.unit), unit_ref(h.unit_ref)
    {
        asm volatile("" : "+s"(starts), "+s"(ends), "+s"(width), "+s"(n), "+s"(unit), "+s"(unit_ref));
    }
};

// A row of up to CM values as they lie in memory, so that the loads of the
// next tile can be in flight while this one is worked on
template <class T, int CM>
struct Packed {
    static constexpr int WORDS = CM * (int)sizeof(T) / 4, PER = 4 / (int)sizeof(T);
    uint32_t w[WORDS];

    template <class W>
    __device__ __forceinline__ void load_units(const char* at, int width)
    {
        constexpr int N = sizeof(W) / 4;
#pragma unroll
        for (int u = 0; u < WORDS / N; u++)
            if (u * N * PER < width) {
                const W t = ((const W*)at)[u];
                __builtin_memcpy(&w[u * N], &t, sizeof(W));
            }
    }
    // `first`: elements from the uniform `rows` to this lane's row; unit: see Small
    __device__ __forceinline__ void load(const T* rows, uint32_t first, int width, int unit)
    {
        const char* at = (const char*)rows + first * (uint32_t)sizeof(T);
        if constexpr (WORDS % 4 == 0) {
            if (unit == 16) return load_units<uint4>(at, width);
        }
        if constexpr (WORDS % 2 == 0) {
            if (unit >= 8) return load_units<uint2>(at, width);
        }
        if (unit >= 4) return load_units<uint32_t>(at, width);
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            T t[PER];
#pragma unroll
            for (int e = 0; e < PER; e++) t[e] = i * PER + e < width ? ((const T*)at)[i * PER + e] : (T)0.f;
            __builtin_memcpy(&w[i], t, 4);
        }
    }
    // -inf behind the row
    __device__ __forceinline__ void get(int width, float* v) const
    {
#pragma unroll
        for (int j = 0; j < CM; j++) {
            const uint32_t u = w[j / PER];
            float f;
            if constexpr (sizeof(T) == 4) f = __builtin_bit_cast(float, u);
            else if constexpr (sizeof(T) == 1) f = (float)(u >> 8 * (j % 4) & 0xffu);
            else if constexpr (__is_same(T, bf16)) f = __builtin_bit_cast(float, j & 1 ? u & 0xffff0000u : u << 16);
            else f = (float)__builtin_bit_cast(f16, (uint16_t)(j & 1 ? u >> 16 : u));
            v[j] = j < width ? f : NEG_INF;
        }
    }
};

template <class T, int CM>
__device__ __forceinline__ void load_row(const T* rows, uint32_t first, int width, int unit, float* v)
{
    Packed<T, CM> p;
    p.load(rows, first, width, unit);
    p.get(width, v);
}

// e^x for drawing: for 16-bit logits 2^(x log2(e)), whose rounded exponent is 2^-20
// near for |x| < 16, far below the logits' own step; for float32 the library's
template <class T>
__device__ __forceinline__ float exp_of(float x)
{
    if constexpr (sizeof(T) == 4) return expf(x);
    return exp2_of(x * LOG2E);
}

__device__ __forceinline__ bool bit(uint64_t b, int j) { return b >> j & 1; }

// v[j] less its head's maximum (0 where a head has no choice; NaN stays)
template <int CM>
__device__ __forceinline__ void subtract_max(const Bounds& h, float* v)
{
    float m[CM];
#pragma unroll
    for (int j = 0; j < CM; j++) m[j] = j == 0 ? v[0] : fmaxf(v[j], bit(h.starts, j) ? NEG_INF : m[j - 1]);
    float top = 0.f;
#pragma unroll
    for (int j = CM - 1; j >= 0; j--) {
        if (bit(h.ends, j)) top = m[j] == NEG_INF ? 0.f : m[j];
        v[j] = v[j] == NEG_INF ? NO_CHOICE : v[j] - top;
    }
}

// row r uses mask row r % mask_rows
__device__ __forceinline__ int64_t mask_row(int64_t mask_rows, int64_t tile_row, uint32_t l)
{
    const int64_t r = tile_row % mask_rows + l;
    return mask_rows >= WAVE ? (r >= mask_rows ? r - mask_rows : r) : (int64_t)((uint32_t)r % (uint32_t)mask_rows);
}

// masked choices to -inf
template <int CM>
__device__ __forceinline__ void apply_mask(const Packed<uint8_t, CM>& m, float* v)
{
#pragma unroll
    for (int j = 0; j < CM; j++) v[j] = (m.w[j / 4] >> 8 * (j % 4) & 0xffu) == 0 ? NEG_INF : v[j];
}

template <class T, int CM>
__global__ __launch_bounds__(256) void sample_narrow_kernel(SampleArgs a, Small h)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t tiles = (a.rows + WAVE - 1) / WAVE, waves = (int64_t)gridDim.x * 4;
    for (int64_t tile = (int64_t)blockIdx.x * 4 + wave; tile < tiles; tile += waves) {
        const Tile at_row(tile, a.rows, lane);
        const bool there = at_row.there;
        const Bounds b(h);
        float v[CM], s[CM];
        load_row<T, CM>((const T*)a.logits + at_row.base * a.ld, at_row.l * (uint32_t)a.ld, h.width, h.unit, v);
        if (a.noise)
            load_row<float, CM>(a.noise + at_row.base * h.width, at_row.l * (uint32_t)h.width, h.width, h.unit_noise, s);
        if (a.mask) {
            Packed<uint8_t, CM> m;
            m.load(a.mask + mask_row(a.mask_rows, at_row.base, at_row.l) * h.width, 0, h.width, h.unit_mask);
            apply_mask<CM>(m, v);
        }
#pragma unroll
        for (int j = 0; j < CM; j++) s[j] = a.noise ? v[j] + s[j] : v[j];
        float raw[CM];
#pragma unroll
        for (int j = 0; j < CM; j++) raw[j] = v[j];
        subtract_max<CM>(b, v);
        float sum = 0.f, t = 0.f, best = NEG_INF, at = __builtin_nanf("");
        int choice = -1, d = 0, first = 0;
        double logp = 0.;
        float entropy = 0.f;
        int32_t* acts = a.actions + at_row.base * h.act_dim;
        const uint32_t act = at_row.l * (uint32_t)h.act_dim;
#pragma unroll
        for (int j = 0; j < CM; j++) {
            const float e = exp_of<T>(v[j]);
            sum += e;
            // (a difference past the largest number: its exponential is 0, not NaN in the product)
            t += e * fmaxf(v[j], -1e30f);
            // the first of the largest scores; a score of -inf counts for a choice that exists
            const bool better = raw[j] != NEG_INF && (s[j] > best || (choice < 0 && s[j] == best));
            best = better ? s[j] : best;
            choice = better ? j : choice;
            at = better ? v[j] : at;
            if (bit(b.ends, j)) {
                const bool some = sum != 0.f;
                const float log_s = some ? log_of(sum) : 0.f;
                logp += some ? (double)at - (double)log_s : 0.;
                entropy += some ? log_s - t * rcp_of(sum) : 0.f;
                if (there) acts[act + h.slot[d]] = h.low[d] + (choice < 0 ? 0 : choice - first);
                sum = t = 0.f;
                best = NEG_INF;
                at = __builtin_nanf("");
                choice = -1;
                first = j + 1;
                d++;
            }
        }
        if (!there) continue;
        if (!h.owned)
            for (int c = 0; c < h.act_dim; c++) {
                bool has = false;
                for (int k = 0; k < h.n; k++) has |= h.slot[k] == c;
                if (!has) acts[act + c] = 0;
            }
        if (a.logp) (a.logp + at_row.base)[at_row.l] = (float)logp;
        if (a.entropy) (a.entropy + at_row.base)[at_row.l] = entropy;
    }
}

// Logits to (logit - top) log2(e), in place: their heads' tops, or, where no
// logit of a wave's rows is more than SPAN below its row's largest, the row's
// (sums of at least 2^(-1.5 SPAN) lose nothing by it): one fma a choice.
constexpr float SPAN = 16.f;

template <int CM>
__device__ __forceinline__ bool row_span(const float* v, int width, float& top)
{
    float low = -NEG_INF;
    top = NEG_INF;
#pragma unroll
    for (int j = 0; j < CM; j++) {
        top = fmaxf(top, v[j]);
        low = fminf(low, j < width ? v[j] : -NEG_INF);
    }
    return low > top - SPAN && fabsf(top) < NEAR_TOP;
}

// the same over the choices that exist
template <int CM>
__device__ __forceinline__ bool some_span(const float* v, float top)
{
    float low = -NEG_INF;
#pragma unroll
    for (int j = 0; j < CM; j++) low = fminf(low, v[j] == NEG_INF ? -NEG_INF : v[j]);
    return top == NEG_INF || (low > top - SPAN && fabsf(top) < NEAR_TOP);
}

template <int CM, bool ALL>
__device__ __forceinline__ void from_row_top(float top, float* v)
{
    const float t = ALL || top != NEG_INF ? -top * LOG2E : 0.f;
#pragma unroll
    for (int j = 0; j < CM; j++) {
        const float x = fmaf(v[j], LOG2E, t);
        v[j] = ALL ? x : v[j] == NEG_INF ? NO_CHOICE : x;
    }
}

template <int CM>
__device__ __forceinline__ void from_head_top(const Bounds& h, float* v)
{
    float m[CM];
#pragma unroll
    for (int j = 0; j < CM; j++) m[j] = j == 0 ? v[0] : fmaxf(v[j], bit(h.starts, j) ? NEG_INF : m[j - 1]);
    float top = 0.f;
#pragma unroll
    for (int j = CM - 1; j >= 0; j--) {
        if (bit(h.ends, j)) top = m[j] == NEG_INF ? 0.f : m[j];
        // a choice 1e30 below the best (masked by its type's lowest value) is as far as any
        const float x = (v[j] - top) * LOG2E;
        v[j] = v[j] == NEG_INF ? NO_CHOICE : x < -1e30f ? -1e30f : x;
    }
}

// The sums of a row's heads lie in LDS, a plane of 64 floats each: every lane
// reads only what it wrote.  The unrolled sweeps over the choices stay short;
// what is done once a head is a loop over the heads.
enum { P_S, P_T, P_AT, P_SR, P_U };             // afterwards 1/S, T/S and 1/S of ref in P_S, P_T, P_SR

template <class T, int CM, bool REF, bool GRAD>
__global__ __launch_bounds__(256) void loss_narrow_kernel(LossArgs a, Small h)
{
    extern __shared__ float4 lds[];
    constexpr int PLANES = REF ? 5 : 3;
    // wide rows' exponentials are made again for the gradient: kept, they cost a third of the waves
    constexpr bool KEEP = GRAD && CM < 32;
    typedef typename std::conditional<(CM > 32), uint64_t, uint32_t>::type Picks;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // per wave: [heads][PLANES][64] sums, then the tile of gradients
    const int tile_bytes = GRAD && h.unit_grad < 0 ? (WAVE * h.width * (int)sizeof(T) + 15) & ~15 : 0;
    char* mine = (char*)lds + wave * (h.n * PLANES * WAVE * 4 + tile_bytes);
    float* planes = (float*)mine + lane;
    T* out = (T*)(mine + h.n * PLANES * WAVE * 4);
    const int64_t tiles = (a.rows + WAVE - 1) / WAVE, waves = (int64_t)gridDim.x * 4;
    float step = 0.f;
    if (GRAD) step = a.scale * (a.upstream ? *a.upstream : 1.f) * inverse_rows(a);
    double sums[N_SUMS] = {0., 0., 0., 0., 0.};
    int64_t clipped = 0, count = 0;
    // what a tile reads, loaded a tile ahead
    struct {
        Packed<T, CM> z, r;
        Packed<uint8_t, CM> mask;
        float adv, old;
        int32_t act[4];
        uint8_t valid;
    } next;
    const auto fetch = [&](int64_t tile) __attribute__((always_inline)) {
        const Tile at_row(tile, a.rows, lane);
        const int64_t base = at_row.base;
        const uint32_t l = at_row.l;
        const Bounds heads(h);
        next.z.load((const T*)a.logits + base * a.ld, l * (uint32_t)a.ld, heads.width, heads.unit);
        if constexpr (REF) next.r.load((const T*)a.ref + base * a.ld_ref, l * (uint32_t)a.ld_ref, heads.width, heads.unit_ref);
        const int32_t* acts = a.actions + base * h.act_dim;
#pragma unroll
        for (int d = 0; d < 4; d++) next.act[d] = acts[l * (uint32_t)h.act_dim + h.slot[d < heads.n ? d : 0]];
        next.adv = (a.advantage + base)[l];
        next.old = (a.old_logp + base)[l];
        next.valid = a.valid ? (a.valid + base)[l] : 1;
        if (a.mask) next.mask.load(a.mask + mask_row(a.mask_rows, base, l) * heads.width, 0, heads.width, h.unit_mask);
    };
    int64_t tile = (int64_t)blockIdx.x * 4 + wave;
    if (tile < tiles) fetch(tile);
    for (; tile < tiles; tile += waves) {
        const Tile at_row(tile, a.rows, lane);
        const int64_t base = at_row.base;
        const uint32_t l = at_row.l;
        const Bounds heads(h);
        float x[CM], y[REF ? CM : 1], e[KEEP ? CM : 1];
        next.z.get(heads.width, x);
        if constexpr (REF) next.r.get(heads.width, y);
        const bool there = at_row.there, valid = there && next.valid;
        const float adv = next.adv, old = next.old;
        // bit j: choice j is its head's action
        Picks picks = 0;
        for (int d = 0; d < heads.n; d += 4) {
            if (d > 0) {
                const int32_t* acts = a.actions + base * h.act_dim;
#pragma unroll
                for (int k = 0; k < 4; k++) next.act[k] = acts[l * (uint32_t)h.act_dim + h.slot[d + k < heads.n ? d + k : 0]];
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t c = (uint32_t)next.act[k] - (uint32_t)h.low[d + k];
                picks |= d + k < heads.n && c < (uint32_t)h.size[d + k] ? (Picks)1 << (h.first[d + k] + (int)c) : 0;
            }
        }
        if (a.mask) apply_mask<CM>(next.mask, x);
        if (tile + waves < tiles) fetch(tile + waves);
        float top, top_r = 0.f;
        bool near = row_span<CM>(x, heads.width, top);
        if constexpr (REF) near &= row_span<CM>(y, heads.width, top_r);
        if (__all(near || !valid)) {
            from_row_top<CM, true>(top, x);
            if constexpr (REF) from_row_top<CM, true>(top_r, y);
        } else {
            near = some_span<CM>(x, top);
            if constexpr (REF) {
#pragma unroll
                for (int j = 0; j < CM; j++) y[j] = x[j] == NEG_INF ? NEG_INF : y[j];
                (void)row_span<CM>(y, heads.width, top_r);
                near &= some_span<CM>(y, top_r);
            }
            if (__all(near || !valid)) {
                from_row_top<CM, false>(top, x);
                if constexpr (REF) from_row_top<CM, false>(top_r, y);
            } else {
                from_head_top<CM>(heads, x);
                if constexpr (REF) from_head_top<CM>(heads, y);
            }
        }
        float s = 0.f, t = 0.f, at = 0.f, sr = 0.f, u = 0.f;
        float* plane = planes;
#pragma unroll
        for (int j = 0; j < CM; j++) {
            const float on = __uint_as_float(0x3f800000u * (1u - (uint32_t)(heads.starts >> j & 1)));
            const float ej = exp2_of(x[j]);
            if constexpr (KEEP) e[j] = ej;
            s = fmaf(on, s, ej);
            t = fmaf(on, t, ej * x[j]);
            const uint32_t pick = 0u - (uint32_t)(picks >> j & 1);
            at = fmaf(on, at, __uint_as_float(pick & __float_as_uint(x[j])));
            if constexpr (REF) {
                const float er = exp2_of(y[j]);
                sr = fmaf(on, sr, er);
                u = fmaf(on, u, er * (y[j] - x[j]));
                if constexpr (KEEP) y[j] = er;
            }
            if (bit(heads.ends, j)) {
                plane[P_S * WAVE] = s;
                plane[P_T * WAVE] = t;
                plane[P_AT * WAVE] = at;
                if constexpr (REF) {
                    plane[P_SR * WAVE] = sr;
                    plane[P_U * WAVE] = u;
                }
                plane += PLANES * WAVE;
            }
        }
        float kl = 0.f, entropy = 0.f;
        double logp = 0.;
        bool possible = true;
        plane = planes;
        for (int d = 0; d < h.n; d++, plane += PLANES * WAVE) {
            const float sd = plane[P_S * WAVE], atd = plane[P_AT * WAVE];
            const bool some = sd != 0.f;
            const float inv = some ? rcp_of(sd) : 0.f, log_s = some ? log_of(sd) : 0.f, ts = plane[P_T * WAVE] * inv;
            const Picks of = ((Picks)~(Picks)0 >> (8 * (int)sizeof(Picks) - h.size[d])) << h.first[d];
            // (NaN, of a NaN or infinite logit there, is found)
            const bool found = (picks & of) != 0 && !(atd <= -1e38f);
            entropy += log_s - ts * LN2;
            possible &= found || !some;
            logp += found && some ? (double)(atd * LN2) - (double)log_s : 0.;
            if constexpr (REF) {
                const float srd = plane[P_SR * WAVE];
                const bool some_ref = some && srd != 0.f;
                const float inv_r = some_ref ? rcp_of(srd) : 0.f;
                kl += some_ref ? plane[P_U * WAVE] * inv_r * LN2 + log_of(sd * inv_r) : 0.f;
                if (GRAD) plane[P_SR * WAVE] = inv_r;
            }
            if (GRAD) {
                plane[P_S * WAVE] = inv;
                plane[P_T * WAVE] = ts;
            }
        }
        const RowLoss r = row_loss(a, adv, old, logp, possible, kl, entropy);
        if (a.logp && there) (a.logp + base)[l] = valid ? r.logp : 0.f;
        if (a.out) {
            sums[S_PG] += valid ? r.pg : 0.f;
            sums[S_KL] += valid ? r.kl : 0.f;
            sums[S_H] += valid ? r.entropy : 0.f;
            clipped += __popcll(__ballot(valid && r.clipped));
            count += __popcll(__ballot(valid));
        }
        if constexpr (GRAD) {
            // g = e/S ((beta - pull) + eta (x - T/S)) - beta er/Sr, and pull at the choice:
            // log p + H = x - T/S
            const float pull = r.pull * step, eta = a.entropy * step * LN2, beta = a.kl * step;
            float a0 = 0.f, a1 = 0.f, b = 0.f;
            const Bounds again(h);
            // products and tests are made again, not kept for every choice
            asm volatile("" : "+v"(picks));
#pragma unroll
            for (int j = 0; j < CM; j++) asm volatile("" : "+v"(x[j]));
            if constexpr (REF && !KEEP)
#pragma unroll
                for (int j = 0; j < CM; j++) asm volatile("" : "+v"(y[j]));
            plane = planes;
#pragma unroll
            for (int j = 0; j < CM; j++) {
                if (bit(again.starts, j)) {
                    const float inv = plane[P_S * WAVE], ts = plane[P_T * WAVE], inv_r = REF ? plane[P_SR * WAVE] : 0.f;
                    a1 = eta * inv;
                    a0 = inv * ((inv_r != 0.f ? beta : 0.f) - pull - eta * ts);
                    b = -beta * inv_r;
                    plane += PLANES * WAVE;
                }
                // (e x is 0 for choices far below, where a1 x may overflow)
                const float ej = KEEP ? e[KEEP ? j : 0] : exp2_of(x[j]);
                float g = fmaf(a1, ej * x[j], ej * a0);
                if constexpr (REF) g = fmaf(b, KEEP ? y[j] : exp2_of(y[j]), g);
                const uint32_t pick = 0u - (uint32_t)(picks >> j & 1);
                g += __uint_as_float(pick & __float_as_uint(pull));
                x[j] = valid && x[j] != NO_CHOICE ? g : 0.f;
            }
            T* grad = (T*)a.grad + base * h.width;
            if (h.unit_grad > 0) {
                // rows of one or two 16-byte pieces: straight from the registers
                if (there) store_row<T, CM>(grad + l * (uint32_t)again.width, again.width, x);
            } else {
                write_tile<T, CM>(out + lane * again.width, again.width, x);
                wave_sync();
                const int64_t rows = a.rows - base < WAVE ? a.rows - base : WAVE;
                copy_tile<T>(out, grad, (int)rows * again.width, h.unit_grad == -16, lane);
                wave_sync();
            }
        }
    }
    if (!a.out) return;
    if (lane == 0) { sums[S_CLIP] = (double)clipped; sums[S_COUNT] = (double)count; }
    block_sums<4>(a, sums);
}

// --------------------------------------------------------- one wide head
// A group of lanes a row: L neighbouring lanes of a wave (several rows a
// wave), or (L = 0) a workgroup of up to 1024 threads.  Each lane holds V
// pieces of 16 bytes of the row in registers, so the maximum, the sums and
// the gradient read the memory once; the gradient makes the exponentials again
// (kept, they would take twice the row's registers and half the waves).
// 4099 rows of 12800 bf16 with ref, loss and gradient: 122 us, 315 MB at 2.6 TB/s;
// 60 us of it are arithmetic, and three rows a CU leave the loads of a row, which
// all come first, uncovered in part.  1024 rows f16 drawn with their noise: 24 us, 79 MB
// at 3.2 TB/s (the bytes: 15 us), by four rows a CU that start together.

// (logit - top) log2(e) of a row, one form for all of its choices: beside a top
// under NEAR_TOP one fma, else the difference first
struct Base {
    float far, shift;
    __device__ __forceinline__ explicit Base(float top)
        : far(fabsf(top) < NEAR_TOP ? 0.f : top), shift(fabsf(top) < NEAR_TOP ? -top * LOG2E : 0.f) {}
    __device__ __forceinline__ float exponent(float z) const { return fmaf(z - far, LOG2E, shift); }
};

template <class T, int V, int L>
struct WideRow {
    static constexpr int PER = 16 / sizeof(T), WORD = 4 / sizeof(T);
    uint32_t w[V * 4];                          // 16-bit logits stay two a register

    // Piece k of this lane is piece at(k) of the row.  The row's last piece is
    // read so that it ends with the row: what it shares with the piece before it
    // is marked as no choice, as is a piece behind the row.
    static __device__ __forceinline__ int at(int k) { return L ? k * L + (threadIdx.x & (L ? L - 1 : 0)) : k * (int)blockDim.x + (int)threadIdx.x; }
    static __device__ __forceinline__ int start(int k, int width) { return at(k) * PER < width - PER ? at(k) * PER : width - PER; }
    // pieces that some lane of this wave has
    static __device__ __forceinline__ int pieces(int width)
    {
        const int step = L ? L : (int)blockDim.x, first = L ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x & ~63);
        int n = 0;
#pragma unroll
        for (int k = 0; k < V; k++) n += (first + k * step) * PER < width ? 1 : 0;
        return n;
    }

    __device__ __forceinline__ float get(int k, int e) const
    {
        const uint32_t u = w[k * 4 + e / WORD];
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, u);
        else if constexpr (__is_same(T, bf16)) return __builtin_bit_cast(float, e & 1 ? u & 0xffff0000u : u << 16);
        else return (float)__builtin_bit_cast(f16, (uint16_t)(e & 1 ? u >> 16 : u));
    }
    __device__ __forceinline__ void none(int k, int e)
    {
        constexpr uint32_t inf = sizeof(T) == 4 ? 0xff800000u : __is_same(T, bf16) ? 0xff80u : 0xfc00u;
        uint32_t& u = w[k * 4 + e / WORD];
        if constexpr (sizeof(T) == 4) u = inf;
        else u = e & 1 ? (u & 0xffffu) | inf << 16 : (u & 0xffff0000u) | inf;
    }
    __device__ __forceinline__ void load(const T* row, int width, int n)
    {
#pragma unroll
        for (int k = 0; k < V; k++)
            if (k < n) __builtin_memcpy(&w[k * 4], row + start(k, width), 16);   // rows may lie anywhere
    }
    __device__ __forceinline__ void ends(int width, int n)
    {
#pragma unroll
        for (int k = 0; k < V; k++) {
            const int over = at(k) * PER - start(k, width);
            if (k < n && over > 0)
#pragma unroll
                for (int e = 0; e < PER; e++)
                    if (e < over) none(k, e);
        }
    }
    __device__ __forceinline__ void mask(const uint8_t* row, int width, int n)
    {
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (k >= n) continue;
            uint8_t m[PER];
            __builtin_memcpy(m, row + start(k, width), PER);
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (!m[e]) none(k, e);
        }
    }
    // choices that the other row has not are none here
    __device__ __forceinline__ void only(const WideRow& o, int n)
    {
#pragma unroll
        for (int k = 0; k < V; k++)
            if (k < n)
#pragma unroll
                for (int e = 0; e < PER; e++)
                    if (o.get(k, e) == NEG_INF) none(k, e);
    }
    // the largest logit, and the smallest (-inf: some choice does not exist)
    __device__ __forceinline__ void range(float& hi, float& lo, int n) const
    {
        hi = NEG_INF;
        lo = -NEG_INF;
#pragma unroll
        for (int k = 0; k < V; k++)
            if (k < n)
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    hi = fmaxf(hi, get(k, e));
                    lo = fminf(lo, get(k, e));
                }
    }
    // The logit's exponent.  PLAIN: every choice exists and all are of ordinary size,
    // top too: one fma.  Whether it is PLAIN may differ between the waves of a row
    // and between the sums and the gradient; the exponent is the same to the bit.
    template <bool PLAIN>
    __device__ __forceinline__ float less(int k, int e, const Base& b) const
    {
        const float z = get(k, e);
        if constexpr (PLAIN) return fmaf(z, LOG2E, b.shift);
        // a choice 1e30 below the best (masked by its type's lowest value) is as far as any
        const float x = b.exponent(z);
        return z == NEG_INF ? NO_CHOICE : x < -1e30f ? -1e30f : x;
    }
    // what was made of the row before is not to be kept beside it: it is made again
    __device__ __forceinline__ void forget()
    {
#pragma unroll
        for (int i = 0; i < V * 4; i++) asm volatile("" : "+v"(w[i]));
    }
};

// sums or maxima of M values over a row's lanes
template <int L, int M, class Op>
__device__ __forceinline__ void over_group(float* v, float (*box)[16], Op op)
{
#pragma unroll
    for (int o = (L ? L : WAVE) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < M; i++) v[i] = op(v[i], __shfl_xor(v[i], o));
    if constexpr (L == 0) {
        const int waves = (int)blockDim.x / WAVE;
        if (waves == 1) return;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < M; i++) box[i][threadIdx.x >> 6] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < M; i++) {
            float t = box[i][0];
            for (int w = 1; w < waves; w++) t = op(t, box[i][w]);
            v[i] = t;
        }
    }
}

struct OneHead { int32_t width, low, slot, act_dim; };

// where a row's lanes are, and which rows they take
template <int L>
struct Rows {
    static constexpr int PER_BLOCK = L ? 256 / (L ? L : 1) : 1;
    static __device__ __forceinline__ int64_t first() { return L ? (int64_t)blockIdx.x * PER_BLOCK + threadIdx.x / (L ? L : 1) : blockIdx.x; }
    static __device__ __forceinline__ bool leader() { return L ? (threadIdx.x & (L ? L - 1 : 0)) == 0 : threadIdx.x == 0; }
};

template <class T, int V, int L>
__global__ __launch_bounds__(L ? 256 : 1024) void sample_wide_kernel(SampleArgs a, OneHead h)
{
    __shared__ float box[2][16];
    __shared__ float best_s[16];
    __shared__ int best_i[16];
    typedef WideRow<T, V, L> Row;
    const int64_t step = (int64_t)gridDim.x * Rows<L>::PER_BLOCK;
    // (a wave's rows go on together: a row behind the last is the last again)
    for (int64_t r0 = (int64_t)blockIdx.x * Rows<L>::PER_BLOCK; r0 < a.rows; r0 += step) {
        const int64_t mine = r0 + (L ? threadIdx.x / (L ? L : 1) : 0), row = mine < a.rows ? mine : a.rows - 1;
        Row z;
        const int pieces = Row::pieces(h.width);
        z.load((const T*)a.logits + row * a.ld, h.width, pieces);
        if (a.mask) z.mask(a.mask + row % a.mask_rows * h.width, h.width, pieces);
        z.ends(h.width, pieces);
        float best = NEG_INF;
        int choice = INT32_MAX;
        const float* noise = a.noise + row * h.width;
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (k >= pieces) continue;
            const int j = Row::start(k, h.width);
            float n[Row::PER];
            if (a.noise) __builtin_memcpy(n, noise + j, sizeof(n));
            else
#pragma unroll
                for (int e = 0; e < Row::PER; e++) n[e] = 0.f;
#pragma unroll
            for (int e = 0; e < Row::PER; e++) {
                const float v = z.get(k, e), s = v + n[e];
                const bool better = v != NEG_INF && (s > best || (choice == INT32_MAX && s == best));
                best = better ? s : best;
                choice = better ? j + e : choice;
            }
        }
        float m[1], low;
        z.range(m[0], low, pieces);
        z.forget();
        const bool whole = low > -1e30f;
        over_group<L, 1>(m, box, [](float p, float q) { return fmaxf(p, q); });
        const float top = m[0] == NEG_INF ? 0.f : m[0];
        const Base base(top);
        float q[2] = {0.f, 0.f};
        const auto sum = [&](auto plain) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (k >= pieces) continue;
#pragma unroll
                for (int e = 0; e < Row::PER; e++) {
                    const float x = z.template less<decltype(plain)::value>(k, e, base), ex = exp2_of(x);
                    q[0] += ex;
                    q[1] += ex * x;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (__all(whole && fabsf(top) < NEAR_TOP)) sum(std::true_type{});
        else sum(std::false_type{});
        q[1] *= LN2;
        over_group<L, 2>(q, box, [](float p, float r) { return p + r; });
#pragma unroll
        for (int o = (L ? L : WAVE) / 2; o > 0; o >>= 1) {
            const float s = __shfl_xor(best, o);
            const int i = __shfl_xor(choice, o);
            if (s > best || (s == best && i < choice)) { best = s; choice = i; }
        }
        if constexpr (L == 0) {
            const int waves = (int)blockDim.x / WAVE;
            if (waves > 1) {
                __syncthreads();
                if ((threadIdx.x & 63) == 0) { best_s[threadIdx.x >> 6] = best; best_i[threadIdx.x >> 6] = choice; }
                __syncthreads();
                for (int w = 0; w < waves; w++)
                    if (best_s[w] > best || (best_s[w] == best && best_i[w] < choice)) { best = best_s[w]; choice = best_i[w]; }
            }
        }
        if (!Rows<L>::leader() || mine >= a.rows) continue;
        const bool some = q[0] != 0.f;
        const int c = choice == INT32_MAX ? 0 : choice;
        int32_t* act = a.actions + row * h.act_dim;
        for (int i = 0; i < h.act_dim; i++) act[i] = i == h.slot ? h.low + c : 0;
        const float log_s = some ? log_of(q[0]) : 0.f;
        // (of the exponent that the sums have, as the loss makes it)
        if (a.logp)
            a.logp[row] = some ? (float)((double)(base.exponent((float)((const T*)a.logits)[row * a.ld + c]) * LN2) - (double)log_s) : 0.f;
        if (a.entropy) a.entropy[row] = some ? log_s - q[1] * rcp_of(q[0]) : 0.f;
    }
}

template <class T, int V, int L, bool REF, bool GRAD>
__global__ __launch_bounds__(L ? 256 : V == 8 ? 512 : 1024) void loss_wide_kernel(LossArgs a, OneHead h)
{
    __shared__ float box[4][16];
    typedef WideRow<T, V, L> Row;
    constexpr int PER = Row::PER;
    double sums[N_SUMS] = {0., 0., 0., 0., 0.};
    float scale = 0.f;
    if (GRAD) scale = a.scale * (a.upstream ? *a.upstream : 1.f) * inverse_rows(a);
    const int64_t step = (int64_t)gridDim.x * Rows<L>::PER_BLOCK;
    for (int64_t r0 = (int64_t)blockIdx.x * Rows<L>::PER_BLOCK; r0 < a.rows; r0 += step) {
        const int64_t mine = r0 + (L ? threadIdx.x / (L ? L : 1) : 0), row = mine < a.rows ? mine : a.rows - 1;
        const bool valid = mine < a.rows && (!a.valid || a.valid[row]);
        const T* zrow = (const T*)a.logits + row * a.ld;
        const uint8_t* mask = a.mask ? a.mask + row % a.mask_rows * h.width : nullptr;
        T* grad = GRAD ? (T*)a.grad + row * h.width : nullptr;
        Row z, r;
        const int pieces = Row::pieces(h.width);
        z.load(zrow, h.width, pieces);
        if constexpr (REF) r.load((const T*)a.ref + row * a.ld_ref, h.width, pieces);
        const int c = (int)((uint32_t)a.actions[row * h.act_dim + h.slot] - (uint32_t)h.low);
        const bool inside = (uint32_t)c < (uint32_t)h.width;
        const float zc = inside && (!mask || mask[c]) ? (float)zrow[c] : NEG_INF;
        if (mask) z.mask(mask, h.width, pieces);
        z.ends(h.width, pieces);
        float m[2] = {NEG_INF, NEG_INF}, q[4] = {0.f, 0.f, 0.f, 0.f}, low, low_r = 0.f;
        z.range(m[0], low, pieces);
        if constexpr (REF) {
            if (__any(low == NEG_INF)) r.only(z, pieces);
            r.range(m[1], low_r, pieces);
            r.forget();
        }
        z.forget();
        over_group<L, REF ? 2 : 1>(m, box, [](float p, float o) { return fmaxf(p, o); });
        const float top = m[0] == NEG_INF ? 0.f : m[0], top_r = m[1] == NEG_INF ? 0.f : m[1];
        const Base base(top), base_r(top_r);
        // (by waves: most rows are plain but for the pieces behind their ends)
        const bool plain_wave = __all(low > -1e30f && low_r > -1e30f && fabsf(top) < NEAR_TOP && fabsf(top_r) < NEAR_TOP);
        const auto sum = [&](auto plain) __attribute__((always_inline)) {
            constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (k >= pieces) continue;
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    const float x = z.template less<PLAIN>(k, e, base), ex = exp2_of(x);
                    q[0] += ex;
                    q[1] += ex * x;
                    if constexpr (REF) {
                        const float y = r.template less<PLAIN>(k, e, base_r), ey = exp2_of(y);
                        q[2] += ey;
                        q[3] += ey * (y - x);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (plain_wave) sum(std::true_type{});
        else sum(std::false_type{});
        over_group<L, REF ? 4 : 2>(q, box, [](float p, float o) { return p + o; });
        const bool some = q[0] != 0.f, some_ref = REF && some && q[2] != 0.f;
        const float inv = some ? rcp_of(q[0]) : 0.f, log_s = some ? log_of(q[0]) : 0.f, ts = q[1] * inv;
        const float inv_r = some_ref ? rcp_of(q[2]) : 0.f;
        const float kl = some_ref ? q[3] * inv_r * LN2 + log_of(q[0] * inv_r) : 0.f;
        const bool found = some && zc != NEG_INF;
        const double logp = found ? (double)(base.exponent(zc) * LN2) - (double)log_s : 0.;
        const RowLoss got = row_loss(a, a.advantage[row], a.old_logp[row], logp, found || !some, kl, log_s - ts * LN2);
        if (Rows<L>::leader() && mine < a.rows) {
            if (a.logp) a.logp[row] = valid ? got.logp : 0.f;
            if (valid) {
                sums[S_PG] += got.pg; sums[S_KL] += got.kl; sums[S_H] += got.entropy;
                sums[S_CLIP] += got.clipped ? 1. : 0.; sums[S_COUNT] += 1.;
            }
        }
        if constexpr (GRAD) {
            z.forget();
            if constexpr (REF) r.forget();
            // e/S ((beta - pull) + eta (x - T/S)) - beta er/Sr, and pull at the choice
            // (log p + H = x - T/S)
            const float pull = got.pull * scale, eta = a.entropy * scale * LN2, beta = a.kl * scale;
            const float a1 = eta * inv, a0 = inv * ((some_ref ? beta : 0.f) - pull - eta * ts), b = -beta * inv_r;
            const auto walk = [&](auto plain) __attribute__((always_inline)) {
                constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    if (k >= pieces) continue;
                    const int j = Row::start(k, h.width), own = Row::at(k) * PER;
                    float g[PER];
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        const float x = z.template less<PLAIN>(k, e, base);
                        g[e] = exp2_of(x) * fmaf(a1, x, a0);
                        if constexpr (REF) g[e] = fmaf(b, exp2_of(r.template less<PLAIN>(k, e, base_r)), g[e]);
                        if (!PLAIN) g[e] = valid && x != NO_CHOICE ? g[e] : 0.f;
                    }
                    if (found && valid && (uint32_t)(c - j) < (uint32_t)PER && c >= own)
#pragma unroll
                        for (int e = 0; e < PER; e++) g[e] += j + e == c ? pull : 0.f;
                    T t[PER];
#pragma unroll
                    for (int e = 0; e < PER; e++) t[e] = (T)g[e];
                    if (mine < a.rows) {
                        if (PLAIN || own == j) __builtin_memcpy(grad + j, t, 16);
                        else
#pragma unroll
                            for (int e = 0; e < PER; e++)
                                if (j + e >= own) grad[j + e] = t[e];
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            if (plain_wave && __all(valid)) walk(std::true_type{});
            else walk(std::false_type{});
        }
    }
    if (!a.out) return;
    if constexpr (L > 0) block_sums<4>(a, sums);
    else if (threadIdx.x < WAVE) block_sums<1>(a, sums);
}

// One row by one workgroup of G threads, as sample_rows_kernel: maximum,
// sums, gradient are three walks over a head (512 rows of 40000 float32 with ref, which
// no group's registers hold: 214 us; drawing them, two walks and the noise: 103 us).
template <class T, int G>
__global__ __launch_bounds__(G) void loss_rows_kernel(LossArgs a, Heads h)
{
    __shared__ float box[G / WAVE];
    extern __shared__ float lds_row[];          // six numbers a head; STAGED: the row (then its gradient), ref's
    constexpr bool STAGED = G == WAVE;
    float *hm = lds_row, *hls = hm + h.n, *hinv = hls + h.n, *hh = hinv + h.n, *hrm = hh + h.n, *hrinv = hrm + h.n;
    float *lz = hrinv + h.n, *lr = lz + h.width;
    Group<G> grp{box};
    const int tid = threadIdx.x;
    const OwnHead own(h, tid < h.n ? tid : 0);
    double sums[N_SUMS] = {0., 0., 0., 0., 0.};
    float step = 0.f;
    if (a.grad) step = a.scale * (a.upstream ? *a.upstream : 1.f) * inverse_rows(a);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        T* g = a.grad ? (T*)a.grad + row * h.width : nullptr;
        if (a.valid && !a.valid[row]) {
            if (g)
                for (int j = tid; j < h.width; j += G) g[j] = (T)0.f;
            if (a.logp && tid == 0) a.logp[row] = 0.f;
            continue;
        }
        const T* z = (const T*)a.logits + row * a.ld;
        const T* zr = a.ref ? (const T*)a.ref + row * a.ld_ref : nullptr;
        const uint8_t* mask = a.mask ? a.mask + (row % a.mask_rows) * h.width : nullptr;
        const int32_t* act = a.actions + row * h.act_dim;
        if constexpr (STAGED) {
            stage_row<T, G>(z, mask, h.width, lz);
            if (zr) stage_row<T, G>(zr, nullptr, h.width, lr);
            __syncthreads();
        }
        const auto logit = [&](int j) __attribute__((always_inline)) { return STAGED ? lz[j] : logit_at(z, mask, j); };
        const auto refs = [&](int j) __attribute__((always_inline)) { return STAGED ? lr[j] : (float)zr[j]; };
        // this lane's heads: their parts of L, KL, H, and how many actions were not possible
        float mine[4] = {0.f, 0.f, 0.f, 0.f};
        for (int d = tid; d < h.n; d += G) {
            const OwnHead at = d == tid ? own : OwnHead(h, d);
            const int lo = at.lo, hi = at.hi;
            if (hi - lo > LANE_HEAD) continue;
            float m = NEG_INF, mr = NEG_INF, s = 0.f, t = 0.f, sr = 0.f, u = 0.f;
            for (int j = lo; j < hi; j++) {
                const float v = logit(j);
                if (v == NEG_INF) continue;
                m = max_nan(m, v);
                if (zr) mr = max_nan(mr, refs(j));
            }
            float log_s = 0.f, inv = 0.f, ent = 0.f, inv_r = 0.f;
            if (m != NEG_INF) {
                for (int j = lo; j < hi; j++) {
                    const float v = logit(j);
                    if (v == NEG_INF) continue;
                    const float x = below(v, m), e = expf(x);
                    s += e;
                    t += e * x;
                    if (zr && refs(j) != NEG_INF) {
                        const float w = below(refs(j), mr), er = expf(w);
                        sr += er;
                        u += er * (w - x);
                    }
                }
                log_s = log_of(s);
                inv = 1.f / s;
                ent = log_s - t * inv;
                mine[2] += ent;
                if (zr && mr != NEG_INF) {
                    inv_r = 1.f / sr;
                    mine[1] += u * inv_r + log_of(s * inv_r);
                }
                const int c = (int)((uint32_t)act[at.slot] - (uint32_t)at.low);
                const float v = c >= 0 && c < hi - lo ? logit(lo + c) : NEG_INF;
                if (v == NEG_INF) mine[3] += 1.f;
                else mine[0] += (v - m) - log_s;
            }
            hm[d] = m; hls[d] = log_s; hinv[d] = inv; hh[d] = ent; hrm[d] = mr; hrinv[d] = inv_r;
        }
        float kl = 0.f, entropy = 0.f;
        double logp = 0.;
        bool possible = true;
        for (int i = 0; i < h.n_large; i++) {
            const int d = h.large[i], lo = h.off[d], hi = h.off[d + 1];
            float m = NEG_INF, mr = NEG_INF;
            for (int j = lo + tid; j < hi; j += G) {
                const float v = logit(j);
                if (v == NEG_INF) continue;
                m = max_nan(m, v);
                if (zr) mr = max_nan(mr, refs(j));
            }
            m = grp.max(m);
            if (zr) mr = grp.max(mr);
            float log_s = 0.f, inv = 0.f, ent = 0.f, inv_r = 0.f;
            if (m != NEG_INF) {
                float s = 0.f, t = 0.f, sr = 0.f, u = 0.f;
                for (int j = lo + tid; j < hi; j += G) {
                    const float v = logit(j);
                    if (v == NEG_INF) continue;
                    const float x = below(v, m), e = expf(x);
                    s += e;
                    t += e * x;
                    if (zr && refs(j) != NEG_INF) {
                        const float w = below(refs(j), mr), er = expf(w);
                        sr += er;
                        u += er * (w - x);
                    }
                }
                s = grp.sum(s);
                t = grp.sum(t);
                log_s = log_of(s);
                inv = 1.f / s;
                ent = log_s - t * inv;
                entropy += ent;
                if (zr && mr != NEG_INF) {
                    sr = grp.sum(sr);
                    u = grp.sum(u);
                    inv_r = 1.f / sr;
                    kl += u * inv_r + log_of(s * inv_r);
                }
                const int c = (int)((uint32_t)act[h.slot[d]] - (uint32_t)h.low[d]);
                const float v = c >= 0 && c < hi - lo ? logit(lo + c) : NEG_INF;
                if (v == NEG_INF) possible = false;
                else logp += (double)(v - m) - (double)log_s;
            }
            if (tid == 0) {
                hm[d] = m; hls[d] = log_s; hinv[d] = inv; hh[d] = ent; hrm[d] = mr; hrinv[d] = inv_r;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) mine[k] = grp.sum(mine[k]);
        const RowLoss r = row_loss(a, a.advantage[row], a.old_logp[row], logp + (double)mine[0], possible && mine[3] == 0.f,
                                   kl + mine[1], entropy + mine[2]);
        if (tid == 0) {
            if (a.logp) a.logp[row] = r.logp;
            sums[S_PG] += r.pg; sums[S_KL] += r.kl; sums[S_H] += r.entropy;
            sums[S_CLIP] += r.clipped ? 1. : 0.; sums[S_COUNT] += 1.;
        }
        if (!g) {
            __syncthreads();                             // the next row's heads go where this one's are
            continue;
        }
        __syncthreads();
        const auto one = [&](int d, int lo, int j, int c) __attribute__((always_inline)) {
            const float v = logit(j);
            float gj = 0.f;
            if (v != NEG_INF) {
                const float x = below(v, hm[d]), p = expf(x) * hinv[d];
                // d(-surrogate) pull (1[chosen] - p), KL p - q, entropy p (log p + H)
                gj = r.pull * ((j - lo == c ? 1.f : 0.f) - p) + a.entropy * p * (x - hls[d] + hh[d]);
                if (hrinv[d] != 0.f) gj += a.kl * (p - expf(refs(j) - hrm[d]) * hrinv[d]);
            }
            if constexpr (STAGED) lz[j] = gj * step;
            else g[j] = (T)(gj * step);
        };
        for (int d = tid; d < h.n; d += G) {
            const OwnHead at = d == tid ? own : OwnHead(h, d);
            const int lo = at.lo, hi = at.hi;
            if (hi - lo > LANE_HEAD) continue;
            const int c = (int)((uint32_t)act[at.slot] - (uint32_t)at.low);
            for (int j = lo; j < hi; j++) one(d, lo, j, c);
        }
        for (int i = 0; i < h.n_large; i++) {
            const int d = h.large[i], lo = h.off[d], hi = h.off[d + 1];
            const int c = (int)((uint32_t)act[h.slot[d]] - (uint32_t)h.low[d]);
            for (int j = lo + tid; j < hi; j += G) one(d, lo, j, c);
        }
        if constexpr (STAGED) {
            __syncthreads();
            for (int j = tid; j < h.width; j += G) g[j] = (T)lz[j];
        }
        __syncthreads();
    }
    if (!a.out || tid >= WAVE) return;
    block_sums<1>(a, sums);
}

constexpr int COUNT_BLOCKS = 256;

// valid rows, counted per block; `wide`: the flags are 16-byte aligned.  5.2 M
// flags take 4.9 us, most of it the launch: the gradient needs 1/M before its first store
__global__ __launch_bounds__(256) void count_kernel(const uint8_t* valid, int64_t rows, int wide, int32_t* counts)
{
    __shared__ int box[4];
    const int64_t pieces = wide ? rows / 16 : 0;
    int n = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
        const uint4 v = ((const uint4*)valid)[i];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // 0x80 in each byte that is not 0
            const uint32_t t = ((w[k] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[k];
            n += __popc(t & 0x80808080u);
        }
    }
    for (int64_t i = pieces * 16 + (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows; i += (int64_t)gridDim.x * 256)
        n += valid[i] != 0;
    n = wave_sum(n);
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = box[0] + box[1] + box[2] + box[3];
}

// the blocks' partial sums, added in a fixed order, to the loss and its parts:
// two waves for each of the sums, eight loads in flight a lane (of 1024 blocks: 4.7 us,
// two round trips to memory)
__global__ __launch_bounds__(2 * N_SUMS * WAVE) void finish_kernel(LossArgs a, int blocks)
{
    __shared__ double box[2 * N_SUMS];
    const int wave = threadIdx.x >> 6, k = wave >> 1;
    const double* p = a.partial + (int64_t)k * blocks;
    double s[8] = {0., 0., 0., 0., 0., 0., 0., 0.};
    for (int b = threadIdx.x & (2 * WAVE - 1); b < blocks; b += 16 * WAVE)
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] += b + i * 2 * WAVE < blocks ? p[b + i * 2 * WAVE] : 0.;
    const double t = wave_sum(((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])));
    if ((threadIdx.x & 63) == 0) box[wave] = t;
    __syncthreads();
    if (threadIdx.x != 0) return;
    double total[N_SUMS];
    for (int i = 0; i < N_SUMS; i++) total[i] = box[2 * i] + box[2 * i + 1];
    write_out(a, total);
}

constexpr int MAX_BLOCKS = 8192;
constexpr int64_t NARROW_BLOCKS = 1024;         // 256 CUs, 4 workgroups of 4 waves each

// the host's heads, checked, as the kernels take them
gw_status take_heads(const gw_policy_heads* p, Heads* h)
{
    LEARN_NEED(p && p->sizes && p->low && p->slots, "heads: null pointer");
    LEARN_NEED(p->n_heads >= 1 && p->n_heads <= GW_MAX_HEADS, "%d heads outside 1..%d", p->n_heads, GW_MAX_HEADS);
    LEARN_NEED(p->act_dim >= 1 && p->act_dim <= 32767, "act_dim %d outside 1..32767", p->act_dim);
    h->n = p->n_heads;
    h->act_dim = p->act_dim;
    h->n_large = 0;
    int64_t w = 0;
    for (int d = 0; d < p->n_heads; d++) {
        LEARN_NEED(p->sizes[d] >= 1, "head %d has %d choices", d, p->sizes[d]);
        LEARN_NEED(p->slots[d] >= 0 && p->slots[d] < p->act_dim, "head %d: column %d outside 0..%d", d,
                   p->slots[d], p->act_dim - 1);
        for (int e = 0; e < d; e++) LEARN_NEED(p->slots[e] != p->slots[d], "heads %d and %d share column %d", e, d, p->slots[d]);
        LEARN_NEED((int64_t)p->low[d] + p->sizes[d] <= (INT64_C(1) << 31), "head %d: values from %d pass int32", d, p->low[d]);
        h->off[d] = (int32_t)w;
        h->low[d] = p->low[d];
        h->slot[d] = (int16_t)p->slots[d];
        if (p->sizes[d] > LANE_HEAD) h->large[h->n_large++] = (int16_t)d;
        w += p->sizes[d];
        LEARN_NEED(w <= (1 << 30), "more than 2^30 choices");
    }
    h->off[p->n_heads] = (int32_t)w;
    h->width = (int32_t)w;
    return GW_OK;
}

int64_t blocks_for(int64_t rows) { return rows < MAX_BLOCKS ? rows : MAX_BLOCKS; }

// the largest piece (a power of two up to 16 bytes) in which rows of this many
// bytes, that far apart, can be read from there
int unit_of(const void* p, int64_t row_bytes, int64_t apart, int64_t rows)
{
    uintptr_t u = (uintptr_t)p | (uintptr_t)row_bytes | (rows > 1 ? (uintptr_t)apart : 0) | 16;
    return (int)(u & -u);
}

// the narrow kernels' heads, or false if the rows are not narrow
bool take_small(const Heads& h, int64_t ld, int64_t ld_ref, Small* s)
{
    // (a tile's offsets are 32 bits)
    if (h.width > NARROW || ld > (1 << 22) || ld_ref > (1 << 22)) return false;
    *s = Small{};
    s->n = h.n; s->act_dim = h.act_dim; s->width = h.width; s->owned = h.n == h.act_dim;
    for (int d = 0; d < h.n; d++) {
        s->starts |= UINT64_C(1) << h.off[d];
        s->ends |= UINT64_C(1) << (h.off[d + 1] - 1);
        s->low[d] = h.low[d];
        s->slot[d] = h.slot[d];
        s->first[d] = (uint8_t)h.off[d];
        s->size[d] = (uint8_t)(h.off[d + 1] - h.off[d]);
    }
    return true;
}

unsigned narrow_blocks(int64_t rows)
{
    const int64_t tiles = (rows + 4 * WAVE - 1) / (4 * WAVE);
    return (unsigned)(tiles < NARROW_BLOCKS ? tiles : NARROW_BLOCKS);
}

template <class T, int CM>
void launch_sample_narrow(const SampleArgs& a, const Small& s, hipStream_t st)
{
    hipLaunchKernelGGL((sample_narrow_kernel<T, CM>), dim3(narrow_blocks(a.rows)), dim3(256), 0, st, a, s);
}

// How a wide head's rows are shared out, or false where registers do not hold
// them: pieces of 16 bytes, one or (from 17 pieces on) four a lane; fewer than a
// wave's lanes a row where the row has fewer pieces.  Four rows' sums then cross a
// wave's lanes in one (65536 rows of 300 bf16, loss and gradient with ref: 64 us, 94
// us with one piece a lane; of 65 f32, 17 pieces: 30 and 38).  Above 1024 pieces the loss
// takes eight a lane: fewer waves a row hold fewer copies of what is not the
// row, so three rows fit a CU in place of two (4099 x 12800 bf16: 8% less time than
// with four; drawing 1024 of them f16, one row and its noise, takes 27 us with eight
// and 24 with four).
struct WideSplit { int v, lanes, threads; };

bool take_wide(const Heads& h, int size, bool loss, WideSplit* w)
{
    if (h.n != 1 || h.width <= NARROW) return false;
    const int64_t bytes = (int64_t)h.width * size;      // (2^30 choices are past 32 bits)
    if (bytes > 16 * 8 * 1024) return false;
    const int pieces = (int)((bytes + 15) / 16);
    w->v = loss && pieces > 1024 ? 8 : pieces > 16 ? 4 : 1;
    const int lanes = (pieces + w->v - 1) / w->v;
    if (lanes > (w->v == 8 ? 512 : 1024)) return false;
    w->lanes = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : lanes <= 64 ? 64 : 0;
    w->threads = w->lanes ? 256 : (lanes + 63) / 64 * 64;
    return true;
}

unsigned wide_blocks(const WideSplit& w, int64_t rows)
{
    // as many as the device holds at once, a few times over
    const int64_t per = w.lanes ? 256 / w.lanes : 1, need = (rows + per - 1) / per;
    const int64_t most = w.lanes ? NARROW_BLOCKS : 4096;
    return (unsigned)(need < most ? need : most);
}

template <class T, int V>
void launch_sample_wide(const SampleArgs& a, const OneHead& o, const WideSplit& w, hipStream_t st)
{
    const dim3 grid(wide_blocks(w, a.rows)), block(w.threads);
    if (w.lanes == 8) hipLaunchKernelGGL((sample_wide_kernel<T, V, 8>), grid, block, 0, st, a, o);
    if (w.lanes == 16) hipLaunchKernelGGL((sample_wide_kernel<T, V, 16>), grid, block, 0, st, a, o);
    if constexpr (V > 1) {
        if (w.lanes == 32) hipLaunchKernelGGL((sample_wide_kernel<T, V, 32>), grid, block, 0, st, a, o);
        if (w.lanes == 64) hipLaunchKernelGGL((sample_wide_kernel<T, V, 64>), grid, block, 0, st, a, o);
        if (w.lanes == 0) hipLaunchKernelGGL((sample_wide_kernel<T, V, 0>), grid, block, 0, st, a, o);
    }
}

template <class T>
void launch_sample(const SampleArgs& a, const Heads& h, hipStream_t st)
{
    WideSplit w;
    if (take_wide(h, sizeof(T), false, &w)) {
        const OneHead o{h.width, h.low[0], h.slot[0], h.act_dim};
        if (w.v == 1) launch_sample_wide<T, 1>(a, o, w, st);
        else launch_sample_wide<T, 4>(a, o, w, st);
        return;
    }
    Small s;
    if (take_small(h, a.rows > 1 ? a.ld : 0, 0, &s)) {
        s.unit = unit_of(a.logits, h.width * sizeof(T), a.ld * sizeof(T), a.rows);
        s.unit_noise = unit_of(a.noise, h.width * 4, h.width * 4, a.rows);
        s.unit_mask = unit_of(a.mask, h.width, h.width, a.rows);
        if (h.width <= 8) launch_sample_narrow<T, 8>(a, s, st);
        else if (h.width <= 16) launch_sample_narrow<T, 16>(a, s, st);
        else if (h.width <= 24) launch_sample_narrow<T, 24>(a, s, st);
        else if (h.width <= 32) launch_sample_narrow<T, 32>(a, s, st);
        else if (h.width <= 40) launch_sample_narrow<T, 40>(a, s, st);
        else launch_sample_narrow<T, 48>(a, s, st);
        return;
    }
    const dim3 grid((unsigned)blocks_for(a.rows));
    if (h.width >= 8192) hipLaunchKernelGGL((sample_rows_kernel<T, 1024>), grid, dim3(1024), 0, st, a, h);
    else if (h.width >= STAGED_ROW) hipLaunchKernelGGL((sample_rows_kernel<T, 256>), grid, dim3(256), 0, st, a, h);
    else hipLaunchKernelGGL((sample_rows_kernel<T, 64>), grid, dim3(64), (a.noise ? 2 : 1) * h.width * 4, st, a, h);
}

template <class T, int CM, bool REF>
void launch_loss_narrow(const LossArgs& a, const Small& s, unsigned blocks, hipStream_t st)
{
    const size_t sums = (size_t)s.n * (REF ? 5 : 3) * WAVE * 4;
    const size_t tile = a.grad && s.unit_grad < 0 ? (WAVE * s.width * sizeof(T) + 15) & ~(size_t)15 : 0, lds = 4 * (sums + tile);
    const auto k = a.grad ? loss_narrow_kernel<T, CM, REF, true> : loss_narrow_kernel<T, CM, REF, false>;
    if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(k, dim3(blocks), dim3(256), lds, st, a, s);
}

template <class T, int CM>
void launch_loss_narrow(const LossArgs& a, const Small& s, unsigned blocks, hipStream_t st)
{
    if (a.ref) launch_loss_narrow<T, CM, true>(a, s, blocks, st);
    else launch_loss_narrow<T, CM, false>(a, s, blocks, st);
}

template <class T, int V, int L>
void launch_loss_wide(const LossArgs& a, const OneHead& o, unsigned blocks, int threads, hipStream_t st)
{
    const dim3 grid(blocks), block(threads);
    if (a.ref && a.grad) hipLaunchKernelGGL((loss_wide_kernel<T, V, L, true, true>), grid, block, 0, st, a, o);
    else if (a.ref) hipLaunchKernelGGL((loss_wide_kernel<T, V, L, true, false>), grid, block, 0, st, a, o);
    else if (a.grad) hipLaunchKernelGGL((loss_wide_kernel<T, V, L, false, true>), grid, block, 0, st, a, o);
    else hipLaunchKernelGGL((loss_wide_kernel<T, V, L, false, false>), grid, block, 0, st, a, o);
}

// returns the number of workgroups, which have left that many partial sums
template <class T>
unsigned launch_loss(const LossArgs& a, const Heads& h, hipStream_t st)
{
    WideSplit w;
    if (take_wide(h, sizeof(T), true, &w)) {
        const OneHead o{h.width, h.low[0], h.slot[0], h.act_dim};
        const unsigned blocks = wide_blocks(w, a.rows);
        if (w.v == 1) {
            if (w.lanes == 8) launch_loss_wide<T, 1, 8>(a, o, blocks, w.threads, st);
            else launch_loss_wide<T, 1, 16>(a, o, blocks, w.threads, st);
        } else if (w.v == 8) launch_loss_wide<T, 8, 0>(a, o, blocks, w.threads, st);
        else if (w.lanes == 8) launch_loss_wide<T, 4, 8>(a, o, blocks, w.threads, st);
        else if (w.lanes == 16) launch_loss_wide<T, 4, 16>(a, o, blocks, w.threads, st);
        else if (w.lanes == 32) launch_loss_wide<T, 4, 32>(a, o, blocks, w.threads, st);
        else if (w.lanes == 64) launch_loss_wide<T, 4, 64>(a, o, blocks, w.threads, st);
        else launch_loss_wide<T, 4, 0>(a, o, blocks, w.threads, st);
        return blocks;
    }
    Small s;
    // LDS for four waves' heads and gradients must fit a CU
    const size_t lds = 4 * (size_t)(h.n * (a.ref ? 5 : 3) * WAVE * 4 + WAVE * h.width * sizeof(T) + 16);
    if (take_small(h, a.rows > 1 ? a.ld : 0, a.rows > 1 ? a.ld_ref : 0, &s) && lds <= 160 * 1024) {
        const unsigned blocks = narrow_blocks(a.rows);
        s.unit = unit_of(a.logits, h.width * sizeof(T), a.ld * sizeof(T), a.rows);
        s.unit_ref = unit_of(a.ref, h.width * sizeof(T), a.ld_ref * sizeof(T), a.rows);
        s.unit_mask = unit_of(a.mask, h.width, h.width, a.rows);
        const bool wide = ((uintptr_t)a.grad & 15) == 0;
        const int64_t row = h.width * sizeof(T);
        s.unit_grad = wide && (row == 16 || row == 32) ? 16 : wide ? -16 : -1;
        if (h.width <= 8) launch_loss_narrow<T, 8>(a, s, blocks, st);
        else if (h.width <= 16) launch_loss_narrow<T, 16>(a, s, blocks, st);
        else if (h.width <= 24) launch_loss_narrow<T, 24>(a, s, blocks, st);
        else if (h.width <= 32) launch_loss_narrow<T, 32>(a, s, blocks, st);
        else if (h.width <= 40) launch_loss_narrow<T, 40>(a, s, blocks, st);
        else launch_loss_narrow<T, 48>(a, s, blocks, st);
        return blocks;
    }
    const unsigned blocks = (unsigned)blocks_for(a.rows);
    const size_t stats = 6 * (size_t)h.n * 4, staged = stats + (a.ref ? 2 : 1) * (size_t)h.width * 4;
    if (h.width >= 8192) hipLaunchKernelGGL((loss_rows_kernel<T, 1024>), dim3(blocks), dim3(1024), stats, st, a, h);
    else if (h.width >= STAGED_ROW) hipLaunchKernelGGL((loss_rows_kernel<T, 256>), dim3(blocks), dim3(256), stats, st, a, h);
    else hipLaunchKernelGGL((loss_rows_kernel<T, 64>), dim3(blocks), dim3(64), staged, st, a, h);
    return blocks;
}

gw_status check_rows(const Heads& h, int32_t dtype, int64_t rows, const void* logits, int64_t ld,
                     const uint8_t* mask, int64_t mask_rows)
{
    LEARN_NEED(dtype >= GW_T_F32 && dtype <= GW_T_BF16, "unknown dtype %d", dtype);
    LEARN_NEED(rows >= 0 && rows <= (INT64_C(1) << 40), "%lld rows", (long long)rows);
    LEARN_NEED(logits || rows == 0, "logits: null pointer");
    LEARN_NEED(ld >= h.width || rows <= 1, "rows of %d logits are %lld apart", h.width, (long long)ld);
    LEARN_NEED(!mask || (mask_rows >= 1 && rows % mask_rows == 0), "%lld mask rows for %lld rows",
               (long long)mask_rows, (long long)rows);
    return GW_OK;
}

}  // namespace

extern "C" {

const char* gw_learn_last_error(void) { return g_err; }
int32_t gw_learn_abi_version(void) { return 1; }

gw_status gw_policy_sample(const gw_policy_heads* heads, int32_t dtype, int64_t n_rows,
                           const void* logits, int64_t ld, const float* noise,
                           const uint8_t* choice_mask, int64_t mask_rows,
                           int32_t* actions, float* logp, float* entropy, void* stream)
{
    Heads h;
    gw_status s = take_heads(heads, &h);
    if (s == GW_OK) s = check_rows(h, dtype, n_rows, logits, ld, choice_mask, mask_rows);
    if (s != GW_OK) return s;
    LEARN_NEED(actions || n_rows == 0, "actions: null pointer");
    if (n_rows == 0) return GW_OK;
    const SampleArgs a{logits, ld, n_rows, noise, choice_mask, mask_rows, actions, logp, entropy};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GW_T_F32) launch_sample<float>(a, h, st);
    else if (dtype == GW_T_F16) launch_sample<f16>(a, h, st);
    else launch_sample<bf16>(a, h, st);
    LEARN_LAUNCHED();
    return GW_OK;
}

int64_t gw_policy_loss_workspace(int64_t n_rows)
{
    (void)n_rows;
    return (int64_t)MAX_BLOCKS * N_SUMS * 8 + COUNT_BLOCKS * 4;
}

gw_status gw_policy_loss(const gw_policy_heads* heads, int32_t dtype, int64_t n_rows,
                         const void* logits, int64_t ld, const void* ref, int64_t ld_ref,
                         const int32_t* actions, const float* advantage, const float* old_logp,
                         const uint8_t* valid, const uint8_t* choice_mask, int64_t mask_rows,
                         float clip_low, float clip_high, float kl_coef, float entropy_coef,
                         float denominator, const float* denominator_at,
                         float grad_scale, const float* upstream,
                         float* loss, float* stats, float* logp, void* grad,
                         void* workspace, int64_t workspace_bytes, void* stream)
{
    Heads h;
    gw_status s = take_heads(heads, &h);
    if (s == GW_OK) s = check_rows(h, dtype, n_rows, logits, ld, choice_mask, mask_rows);
    if (s != GW_OK) return s;
    LEARN_NEED(n_rows == 0 || (actions && advantage && old_logp), "actions, advantage or old_logp: null pointer");
    LEARN_NEED(!ref || ld_ref >= h.width || n_rows <= 1, "rows of %d ref logits are %lld apart", h.width, (long long)ld_ref);
    LEARN_NEED(clip_low >= 0.f && clip_high >= 0.f && isfinite(clip_low) && isfinite(clip_high),
               "clip %g, %g: finite and not negative", clip_low, clip_high);
    LEARN_NEED(isfinite(kl_coef) && isfinite(entropy_coef) && isfinite(grad_scale) && isfinite(denominator),
               "a coefficient is not finite");
    LEARN_NEED(!loss == !stats, "loss and stats: both or neither");
    LEARN_NEED(loss || logp || grad || n_rows == 0, "nothing to compute: loss, logp and grad are null");
    LEARN_NEED(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= gw_policy_loss_workspace(n_rows),
               "workspace: %lld bytes, 8-byte aligned, are needed", (long long)gw_policy_loss_workspace(n_rows));
    const hipStream_t st = (hipStream_t)stream;
    LossArgs a{};
    a.logits = logits; a.ref = kl_coef == 0.f && !loss ? nullptr : ref; a.ld = ld; a.ld_ref = ld_ref; a.rows = n_rows;
    a.actions = actions; a.advantage = advantage; a.old_logp = old_logp;
    a.valid = valid; a.mask = choice_mask; a.mask_rows = mask_rows;
    a.lo = 1.f - clip_low; a.hi = 1.f + clip_high; a.kl = kl_coef; a.entropy = entropy_coef;
    a.denominator = denominator; a.denominator_at = denominator_at;
    a.scale = grad_scale; a.upstream = upstream;
    a.out = loss; a.stats = stats; a.logp = logp; a.grad = grad;
    a.partial = (double*)workspace;
    if (n_rows == 0) {
        if (loss) hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(2 * N_SUMS * WAVE), 0, st, a, 0);
        LEARN_LAUNCHED();
        return GW_OK;
    }
    if (grad && valid && !(denominator > 0.f) && !denominator_at) {
        int32_t* counts = (int32_t*)((double*)workspace + (int64_t)MAX_BLOCKS * N_SUMS);
        const int64_t blocks = (n_rows + 4095) / 4096;
        a.n_counts = (int32_t)(blocks < COUNT_BLOCKS ? blocks : COUNT_BLOCKS);
        a.counts = counts;
        hipLaunchKernelGGL(count_kernel, dim3(a.n_counts), dim3(256), 0, st, valid, n_rows,
                           (int)(((uintptr_t)valid & 15) == 0), counts);
    }
    const unsigned blocks = dtype == GW_T_F32 ? launch_loss<float>(a, h, st)
                          : dtype == GW_T_F16 ? launch_loss<f16>(a, h, st) : launch_loss<bf16>(a, h, st);
    if (loss && blocks > 1) hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(2 * N_SUMS * WAVE), 0, st, a, (int)blocks);
    LEARN_LAUNCHED();
    return GW_OK;
}

}  // extern "C"
