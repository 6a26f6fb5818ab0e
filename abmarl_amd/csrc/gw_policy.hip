// gw_policy.hip — drawing actions from a policy's logits, and the clipped
// policy loss with its gradient (include/gw_learn.h gw_policy_*).
#include <stdarg.h>
#include <stdio.h>

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
};

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
    float* out; float* logp; void* grad;
    const int32_t* counts; int32_t n_counts;    // valid rows per block of count_kernel
    double* partial;                            // [blocks][N_SUMS]
};

enum { S_PG, S_KL, S_H, S_CLIP, S_COUNT, N_SUMS };

// ------------------------------------------------------------ group of G threads
template <int G>
struct Group {
    float* box;                                 // G / 64 floats of LDS
    __device__ float max(float v)
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
    __device__ float sum(float v)
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

template <class T>
__device__ inline float logit_at(const T* row, const uint8_t* mask, int j)
{
    return (mask && !mask[j]) ? NEG_INF : (float)row[j];
}

// One row by one workgroup of G threads, the choices of a head strided over
// them.  Right for every layout: any number of heads, any width.
template <class T, int G>
__global__ __launch_bounds__(G) void sample_rows_kernel(SampleArgs a, Heads h)
{
    __shared__ float box[G / WAVE];
    __shared__ float best_s[G / WAVE];
    __shared__ int best_i[G / WAVE];
    Group<G> grp{box};
    const int tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* z = (const T*)a.logits + row * a.ld;
        const float* noise = a.noise ? a.noise + row * h.width : nullptr;
        const uint8_t* mask = a.mask ? a.mask + (row % a.mask_rows) * h.width : nullptr;
        int32_t* act = a.actions + row * h.act_dim;
        for (int c = tid; c < h.act_dim; c += G) {
            bool owned = false;
            for (int d = 0; d < h.n; d++) owned |= h.slot[d] == c;
            if (!owned) act[c] = 0;
        }
        float logp = 0.f, entropy = 0.f;
        for (int d = 0; d < h.n; d++) {
            const int lo = h.off[d], hi = h.off[d + 1];
            float m = NEG_INF, bs = NEG_INF;
            int bi = INT32_MAX;
            for (int j = lo + tid; j < hi; j += G) {
                const float v = logit_at(z, mask, j);
                if (v == NEG_INF) continue;
                m = max_nan(m, v);
                const float s = noise ? v + noise[j] : v;
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
                const float v = logit_at(z, mask, j);
                if (v == NEG_INF) continue;
                const float e = expf(v - m);
                s += e;
                t += e * (v - m);
            }
            s = grp.sum(s);
            t = grp.sum(t);
            const float log_s = logf(s);
            logp += (logit_at(z, mask, bi) - m) - log_s;
            entropy += log_s - t / s;
            if (tid == 0) act[h.slot[d]] = h.low[d] + (bi - lo);
        }
        if (tid == 0) {
            if (a.logp) a.logp[row] = logp;
            if (a.entropy) a.entropy[row] = entropy;
        }
    }
}

// what a row's loss needs besides its heads' softmax
struct RowLoss {
    float logp, pull, pg, kl, entropy;          // pull: d(-surrogate)/dL = -ratio A where not clipped
    bool clipped;
};

__device__ inline RowLoss row_loss(const LossArgs& a, int64_t row, float logp, bool possible, float kl, float entropy)
{
    RowLoss r;
    r.logp = possible ? logp : NEG_INF;
    const float adv = a.advantage[row];
    const float ratio = possible ? expf(logp - a.old_logp[row]) : 0.f;
    const float clamped = fminf(fmaxf(ratio, a.lo), a.hi);
    const float free = ratio * adv, held = (ratio != ratio ? ratio : clamped) * adv;
    r.clipped = held < free;
    r.pull = r.clipped ? 0.f : -free;
    r.pg = r.clipped ? -held : -free;
    r.kl = kl;
    r.entropy = entropy;
    return r;
}

// 1/M, or 0 where there is nothing to take a mean of
__device__ inline float inverse_rows(const LossArgs& a)
{
    if (a.denominator > 0.f) return 1.f / a.denominator;
    float m;
    if (a.denominator_at) m = *a.denominator_at;
    else if (a.counts) {
        int64_t n = 0;
        for (int i = 0; i < a.n_counts; i++) n += a.counts[i];
        m = (float)n;
    } else m = (float)a.rows;
    return m > 0.f ? 1.f / m : 0.f;
}

// the blocks' sums to the six numbers of gw_policy_loss's out
__device__ inline void write_out(const LossArgs& a, const double* s)
{
    const float given = a.denominator > 0.f ? a.denominator : a.denominator_at ? *a.denominator_at : -1.f;
    const double m = given >= 0.f ? (double)given : s[S_COUNT];
    const double inv = m > 0. ? 1. / m : 0.;
    a.out[0] = (float)((s[S_PG] + (double)a.kl * s[S_KL] - (double)a.entropy * s[S_H]) * inv);
    a.out[1] = (float)(s[S_PG] * inv);
    a.out[2] = (float)(s[S_KL] * inv);
    a.out[3] = (float)(s[S_H] * inv);
    a.out[4] = (float)(s[S_CLIP] * inv);
    a.out[5] = (float)m;
}

// One row by one workgroup of G threads, as sample_rows_kernel: maximum,
// sums, gradient are three walks over a head.
template <class T, int G>
__global__ __launch_bounds__(G) void loss_rows_kernel(LossArgs a, Heads h)
{
    __shared__ float box[G / WAVE];
    __shared__ float hm[GW_MAX_HEADS], hls[GW_MAX_HEADS], hinv[GW_MAX_HEADS], hh[GW_MAX_HEADS],
        hrm[GW_MAX_HEADS], hrinv[GW_MAX_HEADS];
    Group<G> grp{box};
    const int tid = threadIdx.x;
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
        float logp = 0.f, kl = 0.f, entropy = 0.f;
        bool possible = true;
        for (int d = 0; d < h.n; d++) {
            const int lo = h.off[d], hi = h.off[d + 1];
            float m = NEG_INF, mr = NEG_INF;
            for (int j = lo + tid; j < hi; j += G) {
                const float v = logit_at(z, mask, j);
                if (v == NEG_INF) continue;
                m = max_nan(m, v);
                if (zr) mr = max_nan(mr, (float)zr[j]);
            }
            m = grp.max(m);
            if (zr) mr = grp.max(mr);
            float log_s = 0.f, inv = 0.f, ent = 0.f, inv_r = 0.f;
            if (m != NEG_INF) {
                float s = 0.f, t = 0.f, sr = 0.f, u = 0.f;
                for (int j = lo + tid; j < hi; j += G) {
                    const float v = logit_at(z, mask, j);
                    if (v == NEG_INF) continue;
                    const float e = expf(v - m);
                    s += e;
                    t += e * (v - m);
                    if (zr && (float)zr[j] != NEG_INF) {
                        const float w = (float)zr[j] - mr, er = expf(w);
                        sr += er;
                        u += er * (w - (v - m));
                    }
                }
                s = grp.sum(s);
                t = grp.sum(t);
                log_s = logf(s);
                inv = 1.f / s;
                ent = log_s - t * inv;
                entropy += ent;
                if (zr && mr != NEG_INF) {
                    sr = grp.sum(sr);
                    u = grp.sum(u);
                    inv_r = 1.f / sr;
                    kl += u * inv_r + (log_s - logf(sr));
                }
                const int c = act[h.slot[d]] - h.low[d];
                const float v = c >= 0 && c < hi - lo ? logit_at(z, mask, lo + c) : NEG_INF;
                if (v == NEG_INF) possible = false;
                else logp += (v - m) - log_s;
            }
            if (tid == 0) {
                hm[d] = m; hls[d] = log_s; hinv[d] = inv; hh[d] = ent; hrm[d] = mr; hrinv[d] = inv_r;
            }
        }
        const RowLoss r = row_loss(a, row, logp, possible, kl, entropy);
        if (tid == 0) {
            if (a.logp) a.logp[row] = r.logp;
            sums[S_PG] += r.pg; sums[S_KL] += r.kl; sums[S_H] += r.entropy;
            sums[S_CLIP] += r.clipped ? 1. : 0.; sums[S_COUNT] += 1.;
        }
        if (!g) continue;
        __syncthreads();
        for (int d = 0; d < h.n; d++) {
            const int lo = h.off[d], hi = h.off[d + 1], c = act[h.slot[d]] - h.low[d];
            for (int j = lo + tid; j < hi; j += G) {
                const float v = logit_at(z, mask, j);
                float gj = 0.f;
                if (v != NEG_INF) {
                    const float x = v - hm[d], p = expf(x) * hinv[d];
                    // d(-surrogate) pull (1[chosen] - p), KL p - q, entropy p (log p + H)
                    gj = r.pull * ((j - lo == c ? 1.f : 0.f) - p) + a.entropy * p * (x - hls[d] + hh[d]);
                    if (hrinv[d] != 0.f) gj += a.kl * (p - expf((float)zr[j] - hrm[d]) * hrinv[d]);
                }
                g[j] = (T)(gj * step);
            }
        }
        __syncthreads();
    }
    if (!a.out || tid != 0) return;
    if (gridDim.x == 1) write_out(a, sums);
    else
        for (int k = 0; k < N_SUMS; k++) a.partial[(int64_t)blockIdx.x * N_SUMS + k] = sums[k];
}

constexpr int COUNT_BLOCKS = 256;

// valid rows, counted per block
__global__ __launch_bounds__(256) void count_kernel(const uint8_t* valid, int64_t rows, int32_t* counts)
{
    __shared__ int box[4];
    const int64_t per = (rows + gridDim.x - 1) / gridDim.x, from = per * blockIdx.x;
    const int64_t to = from + per < rows ? from + per : rows;
    int n = 0;
    for (int64_t i = from + threadIdx.x; i < to; i += 256) n += valid[i] != 0;
    n = wave_sum(n);
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = box[0] + box[1] + box[2] + box[3];
}

// the blocks' partial sums, added in a fixed order, to the loss and its parts
__global__ __launch_bounds__(256) void finish_kernel(LossArgs a, int blocks)
{
    __shared__ double box[4][N_SUMS];
    double s[N_SUMS] = {0., 0., 0., 0., 0.};
    for (int b = threadIdx.x; b < blocks; b += 256)
        for (int k = 0; k < N_SUMS; k++) s[k] += a.partial[(int64_t)b * N_SUMS + k];
    for (int k = 0; k < N_SUMS; k++) s[k] = wave_sum(s[k]);
    if ((threadIdx.x & 63) == 0)
        for (int k = 0; k < N_SUMS; k++) box[threadIdx.x >> 6][k] = s[k];
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 4; w++)
        for (int k = 0; k < N_SUMS; k++) s[k] += box[w][k];
    write_out(a, s);
}

constexpr int MAX_BLOCKS = 8192;

// the host's heads, checked, as the kernels take them
gw_status take_heads(const gw_policy_heads* p, Heads* h)
{
    LEARN_NEED(p && p->sizes && p->low && p->slots, "heads: null pointer");
    LEARN_NEED(p->n_heads >= 1 && p->n_heads <= GW_MAX_HEADS, "%d heads outside 1..%d", p->n_heads, GW_MAX_HEADS);
    LEARN_NEED(p->act_dim >= 1 && p->act_dim <= 32767, "act_dim %d outside 1..32767", p->act_dim);
    h->n = p->n_heads;
    h->act_dim = p->act_dim;
    int64_t w = 0;
    for (int d = 0; d < p->n_heads; d++) {
        LEARN_NEED(p->sizes[d] >= 1, "head %d has %d choices", d, p->sizes[d]);
        LEARN_NEED(p->slots[d] >= 0 && p->slots[d] < p->act_dim, "head %d: column %d outside 0..%d", d,
                   p->slots[d], p->act_dim - 1);
        for (int e = 0; e < d; e++) LEARN_NEED(p->slots[e] != p->slots[d], "heads %d and %d share column %d", e, d, p->slots[d]);
        h->off[d] = (int32_t)w;
        h->low[d] = p->low[d];
        h->slot[d] = (int16_t)p->slots[d];
        w += p->sizes[d];
        LEARN_NEED(w <= (1 << 30), "more than 2^30 choices");
    }
    h->off[p->n_heads] = (int32_t)w;
    h->width = (int32_t)w;
    return GW_OK;
}

int64_t blocks_for(int64_t rows) { return rows < MAX_BLOCKS ? rows : MAX_BLOCKS; }

template <class T>
void launch_sample(const SampleArgs& a, const Heads& h, hipStream_t st)
{
    const dim3 grid((unsigned)blocks_for(a.rows));
    if (h.width >= 1024) hipLaunchKernelGGL((sample_rows_kernel<T, 256>), grid, dim3(256), 0, st, a, h);
    else hipLaunchKernelGGL((sample_rows_kernel<T, 64>), grid, dim3(64), 0, st, a, h);
}

template <class T>
void launch_loss(const LossArgs& a, const Heads& h, unsigned blocks, hipStream_t st)
{
    if (h.width >= 1024) hipLaunchKernelGGL((loss_rows_kernel<T, 256>), dim3(blocks), dim3(256), 0, st, a, h);
    else hipLaunchKernelGGL((loss_rows_kernel<T, 64>), dim3(blocks), dim3(64), 0, st, a, h);
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
                         float* out, float* logp, void* grad,
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
    LEARN_NEED(out || logp || grad || n_rows == 0, "nothing to compute: out, logp and grad are null");
    LEARN_NEED(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= gw_policy_loss_workspace(n_rows),
               "workspace: %lld bytes, 8-byte aligned, are needed", (long long)gw_policy_loss_workspace(n_rows));
    const hipStream_t st = (hipStream_t)stream;
    LossArgs a{};
    a.logits = logits; a.ref = kl_coef == 0.f && !out ? nullptr : ref; a.ld = ld; a.ld_ref = ld_ref; a.rows = n_rows;
    a.actions = actions; a.advantage = advantage; a.old_logp = old_logp;
    a.valid = valid; a.mask = choice_mask; a.mask_rows = mask_rows;
    a.lo = 1.f - clip_low; a.hi = 1.f + clip_high; a.kl = kl_coef; a.entropy = entropy_coef;
    a.denominator = denominator; a.denominator_at = denominator_at;
    a.scale = grad_scale; a.upstream = upstream;
    a.out = out; a.logp = logp; a.grad = grad;
    a.partial = (double*)workspace;
    if (n_rows == 0) {
        if (out) hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(256), 0, st, a, 0);
        LEARN_LAUNCHED();
        return GW_OK;
    }
    if (grad && valid && !(denominator > 0.f) && !denominator_at) {
        int32_t* counts = (int32_t*)((double*)workspace + (int64_t)MAX_BLOCKS * N_SUMS);
        const int64_t blocks = (n_rows + 4095) / 4096;
        a.n_counts = (int32_t)(blocks < COUNT_BLOCKS ? blocks : COUNT_BLOCKS);
        a.counts = counts;
        hipLaunchKernelGGL(count_kernel, dim3(a.n_counts), dim3(256), 0, st, valid, n_rows, counts);
    }
    const unsigned blocks = (unsigned)blocks_for(n_rows);
    if (dtype == GW_T_F32) launch_loss<float>(a, h, blocks, st);
    else if (dtype == GW_T_F16) launch_loss<f16>(a, h, blocks, st);
    else launch_loss<bf16>(a, h, blocks, st);
    if (out && blocks > 1) hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(256), 0, st, a, (int)blocks);
    LEARN_LAUNCHED();
    return GW_OK;
}

}  // extern "C"
