// gw_recurrence.hip — the gated linear recurrence over the steps of a
// fragment, its gradients, and the advantages it gives over a rollout's slabs
// (include/gw_learn.h gw_recurrence*, gw_advantages, gw_fragment_marks).
#include "gw_learn.hpp"

namespace {

constexpr int SEG = GW_RECURRENCE_SEGMENT;

struct RecurArgs {
    int64_t T, n;
    const void* x; const void* gate; int64_t gate_span; float gate_value;
    const uint8_t* cut; int64_t cut_span;
    const float* state; int32_t reverse;
    void* h; float* last; float* carry;          // forward
    const void* dh; const float* dlast;          // backward
    void* dx; void* dgate; float* dstate;
    float* part; int32_t parts;                  // [T][n / gate_span][parts]: shared gates' gradients
};

// step i of the recurrence's own order is step at(i) of the slabs
__device__ inline int64_t step_at(const RecurArgs& a, int64_t i) { return a.reverse ? a.T - 1 - i : i; }

template <class TG>
__device__ inline float gate_at(const RecurArgs& a, int64_t t, int64_t c)
{
    if (a.cut && a.cut[t * (a.n / a.cut_span) + c / a.cut_span]) return 0.f;
    return a.gate ? (float)((const TG*)a.gate)[t * (a.n / a.gate_span) + c / a.gate_span] : a.gate_value;
}

// a cut step's state is not used at all: 0 * inf would be NaN
__device__ inline float advance(float gate, float h, float x) { return (gate == 0.f ? 0.f : gate * h) + x; }

// One thread per channel, the steps one after another.
template <class T, class TG>
__global__ __launch_bounds__(256) void recur_kernel(RecurArgs a)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.n) return;
    float h = a.state ? a.state[c] : 0.f;
    for (int64_t i = 0; i < a.T; i++) {
        const int64_t t = step_at(a, i);
        if (a.carry && i % SEG == 0) a.carry[i / SEG * a.n + c] = h;
        h = advance(gate_at<TG>(a, t, c), h, (float)((const T*)a.x)[t * a.n + c]);
        ((T*)a.h)[t * a.n + c] = (T)h;
    }
    if (a.last) a.last[c] = h;
}

// One thread per channel; the segments from the last to the first: the state
// before each step again from the segment's carry, then the steps backwards.
template <class T, class TG>
__global__ __launch_bounds__(64) void recur_backward_kernel(RecurArgs a)
{
    // a wave holds channels of one gate only, so its sum is one gate's part
    // (a gate of its own for each channel: all of them are one group)
    const int64_t span = a.gate_span == 1 ? a.n : a.gate_span;
    const int64_t per = (span + 63) / 64;
    const int64_t group = blockIdx.x / per, piece = blockIdx.x % per;
    const int64_t in = piece * 64 + threadIdx.x;
    const bool on = in < span;
    const int64_t c = group * span + (on ? in : 0);
    float into = on && a.dlast ? a.dlast[c] : 0.f;       // what the next step hands back
    for (int64_t s = (a.T + SEG - 1) / SEG; s-- > 0;) {
        const int64_t i0 = s * SEG;
        const int m = a.T - i0 < SEG ? (int)(a.T - i0) : SEG;
        float before[SEG];
        float h = a.carry[s * a.n + c];
        for (int k = 0; k < m; k++) {
            const int64_t t = step_at(a, i0 + k);
            before[k] = h;
            h = advance(gate_at<TG>(a, t, c), h, (float)((const T*)a.x)[t * a.n + c]);
        }
        for (int k = m - 1; k >= 0; k--) {
            const int64_t t = step_at(a, i0 + k);
            const float g = into + (a.dh ? (float)((const T*)a.dh)[t * a.n + c] : 0.f);
            const float gate = gate_at<TG>(a, t, c);
            into = gate == 0.f ? 0.f : gate * g;
            if (on) ((T*)a.dx)[t * a.n + c] = (T)g;
            if (!a.dgate) continue;
            const bool cut = a.cut && a.cut[t * (a.n / a.cut_span) + c / a.cut_span];
            float d = cut || !on ? 0.f : g * before[k];
            if (a.gate_span == 1) {
                if (on) ((TG*)a.dgate)[t * a.n + c] = (TG)d;
            } else {
                d = wave_sum(d);
                if (threadIdx.x == 0) a.part[(t * (a.n / a.gate_span) + group) * a.parts + piece] = d;
            }
        }
    }
    if (on && a.dstate) a.dstate[c] = into;
}

template <class TG>
__global__ __launch_bounds__(256) void gate_parts_kernel(const float* part, int parts, int64_t gates, TG* dgate)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= gates) return;
    float s = 0.f;
    for (int p = 0; p < parts; p++) s += part[i * parts + p];
    dgate[i] = (TG)s;
}

__global__ __launch_bounds__(256) void marks_kernel(int64_t T, int64_t E, const uint8_t* all_done,
                                                    const uint8_t* all_done_in, const int32_t* steps,
                                                    const uint32_t* err, int32_t horizon, int32_t mode, uint8_t* marks)
{
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= E) return;
    int64_t n = steps ? steps[e] : 0;
    bool ended = all_done_in && all_done_in[e];
    const uint8_t skip = err && err[e] ? GW_MARK_SKIP : 0;
    for (int64_t t = 0; t < T; t++) {
        uint8_t m = skip;
        if (mode == 2 && (ended || (horizon > 0 && n >= horizon))) {
            m |= GW_MARK_RESET;
            n = 0;
            ended = false;
        } else {
            n += 1;
            ended = all_done[t * E + e] != 0;
            const bool horizon_hit = horizon > 0 && n >= horizon;
            if (ended || (mode == 1 && horizon_hit)) m |= GW_MARK_END;
            else if (horizon_hit) m |= GW_MARK_TRUNCATED;
            if (mode == 1 && (ended || horizon_hit)) n = 0;
        }
        marks[t * E + e] = m;
    }
}

struct AdvArgs {
    int64_t T, E, A;
    const void* reward; const void* value; const uint8_t* done; const uint8_t* marks; const uint8_t* live;
    const uint8_t* acts;
    float gamma, lam;
    float* advantage; float* target; uint8_t* valid;
};

// whether the lane acted in step t
__device__ inline bool acted(const AdvArgs& a, int64_t t, int64_t c, int64_t e, uint8_t mark)
{
    if (mark & (GW_MARK_RESET | GW_MARK_SKIP)) return false;
    if (a.acts && !a.acts[c % a.A]) return false;
    if (t == 0) return a.live[c] != 0;
    return (a.marks[(t - 1) * a.E + e] & GW_MARK_END) || !a.done[(t - 1) * a.E * a.A + c];
}

template <class TR, class TV>
__global__ __launch_bounds__(256) void advantages_kernel(AdvArgs a)
{
    const int64_t n = a.E * a.A, c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    const int64_t e = c / a.A;
    float carry = 0.f;
    for (int64_t t = a.T; t-- > 0;) {
        const int64_t i = t * n + c;
        const uint8_t mark = a.marks[t * a.E + e];
        const bool ok = acted(a, t, c, e, mark);
        float target = 0.f;
        if (ok) {
            const bool final = a.done[i] || (mark & GW_MARK_END);
            const float v = (float)((const TV*)a.value)[i];
            float d = (float)((const TR*)a.reward)[i] - v;
            if (!final) {
                d += a.gamma * (float)((const TV*)a.value)[i + n];
                if (!(mark & GW_MARK_TRUNCATED)) d += a.gamma * a.lam * carry;
            }
            carry = d;
            target = d + v;
        } else {
            carry = 0.f;
        }
        a.advantage[i] = carry;
        a.target[i] = target;
        a.valid[i] = ok;
    }
}

template <class T, class TG>
void launch_recurrence(const RecurArgs& a, hipStream_t st)
{
    hipLaunchKernelGGL((recur_kernel<T, TG>), dim3((unsigned)((a.n + 255) / 256)), dim3(256), 0, st, a);
}

template <class T, class TG>
void launch_backward(const RecurArgs& a, hipStream_t st)
{
    const int64_t gates = a.n / a.gate_span;
    const int64_t span = a.gate_span == 1 ? a.n : a.gate_span;
    hipLaunchKernelGGL((recur_backward_kernel<T, TG>), dim3((unsigned)(a.n / span * ((span + 63) / 64))), dim3(64), 0,
                       st, a);
    if (a.dgate && a.gate_span > 1)
        hipLaunchKernelGGL((gate_parts_kernel<TG>), dim3((unsigned)((a.T * gates + 255) / 256)), dim3(256), 0, st,
                           a.part, a.parts, a.T * gates, (TG*)a.dgate);
}

gw_status check_recurrence(int32_t dtype, int32_t gate_dtype, int64_t T, int64_t n, const void* x, const void* gate,
                           int64_t gate_span, float gate_value, const uint8_t* cut, int64_t cut_span)
{
    LEARN_NEED(dtype >= GW_T_F32 && dtype <= GW_T_BF16, "unknown dtype %d", dtype);
    LEARN_NEED(gate_dtype == dtype || gate_dtype == GW_T_F32, "gate_dtype %d with dtype %d: the same or GW_T_F32",
               gate_dtype, dtype);
    LEARN_NEED(T >= 0 && n >= 0 && T <= (INT64_C(1) << 31) && n <= (INT64_C(1) << 31), "%lld steps of %lld channels",
               (long long)T, (long long)n);
    LEARN_NEED(T == 0 || n == 0 || x, "x: null pointer");
    LEARN_NEED(gate_span >= 1 && n % gate_span == 0, "gate_span %lld for %lld channels", (long long)gate_span, (long long)n);
    LEARN_NEED(gate || isfinite(gate_value), "gate_value is not finite");
    LEARN_NEED(!cut || (cut_span >= 1 && n % cut_span == 0), "cut_span %lld for %lld channels", (long long)cut_span,
               (long long)n);
    return GW_OK;
}

int64_t gate_pieces(int64_t gate_span) { return (gate_span + 63) / 64; }

}  // namespace

extern "C" {

int64_t gw_recurrence_workspace(int64_t n_steps, int64_t n)
{
    (void)n_steps; (void)n;
    return 0;
}

gw_status gw_recurrence(int32_t dtype, int32_t gate_dtype, int64_t n_steps, int64_t n,
                        const void* x, const void* gate, int64_t gate_span, float gate_value,
                        const uint8_t* cut, int64_t cut_span, const float* state, int32_t reverse,
                        void* h, float* last, float* carry,
                        void* workspace, int64_t workspace_bytes, void* stream)
{
    (void)workspace; (void)workspace_bytes;
    const gw_status s = check_recurrence(dtype, gate_dtype, n_steps, n, x, gate, gate_span, gate_value, cut, cut_span);
    if (s != GW_OK) return s;
    LEARN_NEED(n_steps == 0 || n == 0 || h, "h: null pointer");
    if (n == 0) return GW_OK;
    RecurArgs a{};
    a.T = n_steps; a.n = n; a.x = x; a.gate = gate; a.gate_span = gate_span; a.gate_value = gate_value;
    a.cut = cut; a.cut_span = cut_span; a.state = state; a.reverse = reverse;
    a.h = h; a.last = last; a.carry = carry;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GW_T_F32) launch_recurrence<float, float>(a, st);
    else if (dtype == GW_T_F16) gate_dtype == dtype ? launch_recurrence<f16, f16>(a, st) : launch_recurrence<f16, float>(a, st);
    else gate_dtype == dtype ? launch_recurrence<bf16, bf16>(a, st) : launch_recurrence<bf16, float>(a, st);
    LEARN_LAUNCHED();
    return GW_OK;
}

int64_t gw_recurrence_backward_workspace(int64_t n_steps, int64_t n, int64_t gate_span)
{
    if (n_steps <= 0 || n <= 0 || gate_span <= 1) return 0;
    return n_steps * (n / gate_span) * gate_pieces(gate_span) * 4;
}

gw_status gw_recurrence_backward(int32_t dtype, int32_t gate_dtype, int64_t n_steps, int64_t n,
                                 const void* x, const void* gate, int64_t gate_span, float gate_value,
                                 const uint8_t* cut, int64_t cut_span, const float* carry, int32_t reverse,
                                 const void* dh, const float* dlast,
                                 void* dx, void* dgate, float* dstate,
                                 void* workspace, int64_t workspace_bytes, void* stream)
{
    const gw_status s = check_recurrence(dtype, gate_dtype, n_steps, n, x, gate, gate_span, gate_value, cut, cut_span);
    if (s != GW_OK) return s;
    LEARN_NEED(n_steps == 0 || n == 0 || (carry && dx), "carry or dx: null pointer");
    LEARN_NEED(!dgate || gate, "dgate without gate");
    const int64_t need = dgate ? gw_recurrence_backward_workspace(n_steps, n, gate_span) : 0;
    LEARN_NEED(need == 0 || (workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need),
               "workspace: %lld bytes, 8-byte aligned, are needed", (long long)need);
    if (n == 0) return GW_OK;
    RecurArgs a{};
    a.T = n_steps; a.n = n; a.x = x; a.gate = gate; a.gate_span = gate_span; a.gate_value = gate_value;
    a.cut = cut; a.cut_span = cut_span; a.reverse = reverse; a.carry = const_cast<float*>(carry);
    a.dh = dh; a.dlast = dlast; a.dx = dx; a.dgate = dgate; a.dstate = dstate;
    a.part = (float*)workspace; a.parts = (int32_t)gate_pieces(gate_span);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GW_T_F32) launch_backward<float, float>(a, st);
    else if (dtype == GW_T_F16) gate_dtype == dtype ? launch_backward<f16, f16>(a, st) : launch_backward<f16, float>(a, st);
    else gate_dtype == dtype ? launch_backward<bf16, bf16>(a, st) : launch_backward<bf16, float>(a, st);
    LEARN_LAUNCHED();
    return GW_OK;
}

gw_status gw_fragment_marks(int64_t n_steps, int64_t n_envs, const uint8_t* all_done,
                            const uint8_t* all_done_in, const int32_t* steps, const uint32_t* err,
                            int32_t horizon, int32_t autoreset, uint8_t* marks, void* stream)
{
    LEARN_NEED(n_steps >= 0 && n_envs >= 0 && n_envs <= (INT64_C(1) << 31), "%lld steps of %lld envs",
               (long long)n_steps, (long long)n_envs);
    LEARN_NEED(autoreset == 1 || autoreset == 2, "autoreset %d: 1 (same step) or 2 (next step)", autoreset);
    LEARN_NEED(n_steps == 0 || n_envs == 0 || (all_done && marks), "all_done or marks: null pointer");
    if (n_steps == 0 || n_envs == 0) return GW_OK;
    hipLaunchKernelGGL(marks_kernel, dim3((unsigned)((n_envs + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                       n_steps, n_envs, all_done, all_done_in, steps, err, horizon, autoreset, marks);
    LEARN_LAUNCHED();
    return GW_OK;
}

gw_status gw_advantages(int32_t dtype, int32_t reward_f64, int64_t n_steps, int64_t n_envs, int64_t n_lanes,
                        const void* reward, const void* value, const uint8_t* done, const uint8_t* marks,
                        const uint8_t* live, const uint8_t* acts, float gamma, float lam,
                        float* advantage, float* target, uint8_t* valid,
                        void* workspace, int64_t workspace_bytes, void* stream)
{
    (void)workspace; (void)workspace_bytes;
    LEARN_NEED(dtype >= GW_T_F32 && dtype <= GW_T_BF16, "unknown dtype %d", dtype);
    LEARN_NEED(n_steps >= 0 && n_envs >= 0 && n_lanes >= 1 && n_envs <= (INT64_C(1) << 31) / n_lanes,
               "%lld steps of %lld envs of %lld lanes", (long long)n_steps, (long long)n_envs, (long long)n_lanes);
    LEARN_NEED(isfinite(gamma) && isfinite(lam), "gamma or lam is not finite");
    if (n_steps == 0 || n_envs == 0) return GW_OK;
    LEARN_NEED(reward && value && done && marks && live && advantage && target && valid, "null pointer");
    const AdvArgs a{n_steps, n_envs, n_lanes, reward, value, done, marks, live, acts, gamma, lam, advantage, target, valid};
    const dim3 grid((unsigned)((n_envs * n_lanes + 255) / 256));
    const hipStream_t st = (hipStream_t)stream;
#define ADV(TR, TV) hipLaunchKernelGGL((advantages_kernel<TR, TV>), grid, dim3(256), 0, st, a)
    if (reward_f64) {
        if (dtype == GW_T_F32) ADV(double, float);
        else if (dtype == GW_T_F16) ADV(double, f16);
        else ADV(double, bf16);
    } else {
        if (dtype == GW_T_F32) ADV(float, float);
        else if (dtype == GW_T_F16) ADV(float, f16);
        else ADV(float, bf16);
    }
#undef ADV
    LEARN_LAUNCHED();
    return GW_OK;
}

}  // extern "C"
