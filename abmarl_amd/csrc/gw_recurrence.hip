// gw_recurrence.hip — the gated linear recurrence over the steps of a
// fragment, its gradients, and the advantages it gives over a rollout's slabs
// (include/gw_learn.h gw_recurrence*, gw_advantages, gw_fragment_marks).
#include "gw_learn.hpp"

namespace {

constexpr int SEG = GW_RECURRENCE_SEGMENT;

struct RecurArgs {
    int64_t T, n;
    const void* x; const void* gate; const uint8_t* cut;
    uint32_t gate_span, cut_span;                // channels per gate, per cut
    int64_t gates, cuts;                         // of a step
    float gate_value;
    const float* state; int32_t reverse;
    void* h; float* last; float* carry;          // forward
    const void* dh; const float* dlast;          // backward
    void* dx; void* dgate; float* dstate;
    float* part; int32_t parts;                  // [T][n / gate_span][parts]: shared gates' gradients
};

// ------------------------------------------------------------------ the scan
// A step is the map h -> a h + b; maps compose, so the steps can be split.  A
// wave holds 64 neighbouring channels (one a lane) and SEG steps of them in
// registers.  NW waves of a workgroup hold NW such segments in time, exchange
// their maps through LDS and walk their own steps from the state that reaches
// them: one pass over the data.  CW waves stand side by side in channels.
// Where channels and waves do not fill the device, the steps are cut into
// chunks too: a first launch makes every chunk's map (reading gates and
// values), a second composes the maps before its own and walks.
//
// Memory bounds long slabs, launches and round trips short ones:
//   20 steps of 1048576 channels bf16, a cut a step: 41 us forward (143 MB, 3.5
//     TB/s) and 48 us backward (227 MB, 4.7 TB/s), by pairs (below);
//   65537 steps of 96 channels f32, a gate a step: maps 12 and 12 us, walks 19 and
//     28 us, parts of the gates' sums 4 us, where 127 MB would take 24 us: a
//     chunk's 8 waves wait for each other's maps, and for those of the chunks before;
//   one step of 262144 channels bf16: 6.9 us, a launch and one round trip.

struct Map { float a, b; };

// A map drops the state only where a gate is 0.  The product of others may
// underflow: then the smallest number keeps an infinite state infinite.
__device__ __forceinline__ float keep(float a, bool zero) { return zero ? 0.f : (a == 0.f ? 1.4e-45f : a); }

// a h + b, where a = 0 drops any state (0 * inf would be NaN)
__device__ __forceinline__ float advance(float a, float h, float b) { return fmaf(a, a == 0.f ? 0.f : h, b); }

// the same for a segment's map, whose product of gates may have overflowed
__device__ __forceinline__ float apply(Map m, float h) { return m.a == 0.f || h == 0.f ? m.b : fmaf(m.a, h, m.b); }

__device__ __forceinline__ Map compose(Map first, Map then)
{
    return Map{keep(first.a * then.a, first.a == 0.f || then.a == 0.f), apply(then, first.b)};
}

// chunks of the steps; maps[chunk][n]
struct Chunks { int32_t count; int64_t steps; float2* maps; };

// The state that reaches wave w's segment, from the one that reaches the
// tile (`in`, which becomes the one behind the tile) and the waves' maps.
template <int NW>
__device__ __forceinline__ float join(float2 (*box)[WAVE], int w, int lane, Map m, float& in)
{
    box[w][lane] = make_float2(m.a, m.b);
    __syncthreads();
    float h = in, mine = in;
#pragma unroll
    for (int v = 0; v < NW; v++) {
        mine = v == w ? h : mine;
        const float2 q = box[v][lane];
        h = apply(Map{q.x, q.y}, h);
    }
    in = h;
    return mine;
}

// The state that reaches a chunk: `state` through the maps of the chunks
// before it, shared out to the NW waves.
template <int NW>
__device__ __forceinline__ float reach_chunk(float2 (*box)[WAVE], const Chunks& s, int64_t n, int64_t c, int w, int lane,
                                    float state)
{
    const int chunk = blockIdx.y;
    if (chunk == 0) return state;
    const int per = (chunk + NW - 1) / NW, from = w * per, to = from + per < chunk ? from + per : chunk;
    Map m{1.f, 0.f};
    for (int j = from; j < to; j += 8) {
        float2 q[8];
#pragma unroll
        for (int k = 0; k < 8; k++) q[k] = s.maps[(int64_t)(j + k < to ? j + k : to - 1) * n + c];
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (j + k < to) m = compose(m, Map{q[k].x, q[k].y});
    }
    if constexpr (NW == 1) return apply(m, state);
    join<NW>(box, w, lane, m, state);
    __syncthreads();
    return state;
}

// Where a wave stands: channels from c0 (uniform), lane l of them (a valid
// one where the lane is not `on`), time segment w of NW.
struct Place {
    int64_t c0;
    int w, lane;
    uint32_t l;
    bool on;
    __device__ __forceinline__ int64_t c() const { return c0 + l; }
};

template <int NW, int CW>
__device__ __forceinline__ Place place(int64_t n)
{
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    Place p;
    p.lane = threadIdx.x & 63;
    p.w = NW == 1 ? 0 : wave;
    p.c0 = ((int64_t)blockIdx.x * CW + (NW == 1 ? wave : 0)) * WAVE;
    const int64_t left = n - 1 - p.c0;
    p.on = p.lane <= left;
    p.l = p.on ? p.lane : 0;
    return p;
}

// A row of one value per `span` channels as the wave's channels see it: from
// a uniform place, per lane a small offset
struct Shared {
    uint32_t first, l;
    __device__ __forceinline__ Shared(uint32_t span, const Place& p)
    {
        // (fewer than 2^31 channels)
        first = (uint32_t)p.c0 / span;
        l = (((uint32_t)p.c0 + p.l) / span - first) & 63u;
    }
};

// step i of the recurrence's own order is step at(i) of the slabs
__device__ __forceinline__ int64_t step_at(const RecurArgs& a, int64_t i) { return a.reverse ? a.T - 1 - i : i; }

// SEG rows of `stride` values from step i0 on, one value a lane: f(k, value).
// Whole segments are one run of loads; in the last one the steps that are
// there are a uniform branch each.
template <class V, class F>
__device__ __forceinline__ void load_rows(const RecurArgs& a, const V* slab, int64_t stride, int64_t i0, int64_t first,
                                 uint32_t l, F f)
{
    const V* row = slab + step_at(a, i0) * stride + first;
    const int64_t next = a.reverse ? -stride : stride;
    V v[SEG];
    if (i0 + SEG <= a.T) {
#pragma unroll
        for (int k = 0; k < SEG; k++, row += next) v[k] = row[l];
#pragma unroll
        for (int k = 0; k < SEG; k++) f(k, v[k]);
    } else {
        const int m = (int)(a.T - i0);
#pragma unroll
        for (int k = 0; k < SEG; k++, row += next)
            if (k < m) f(k, row[l]);
    }
}

// The gates of SEG steps from i0 (0 where cut; 1 behind the last step), and
// cuts as bits
template <class TG>
__device__ __forceinline__ uint32_t load_gates(const RecurArgs& a, int64_t i0, const Shared& g, const Shared& c, float* gate)
{
    uint32_t bits = 0;
    const int m = i0 + SEG <= a.T ? SEG : (int)(a.T - i0);
#pragma unroll
    for (int k = 0; k < SEG; k++) gate[k] = k < m ? a.gate_value : 1.f;
    if (a.gate) load_rows(a, (const TG*)a.gate, a.gates, i0, g.first, g.l, [&](int k, TG v) { gate[k] = (float)v; });
    if (a.cut)
        load_rows(a, a.cut, a.cuts, i0, c.first, c.l, [&](int k, uint8_t v) {
            bits |= (v ? 1u : 0u) << k;
            gate[k] = v ? 0.f : gate[k];
        });
    return bits;
}

// SEG steps of a slab like x; 0 behind the last step
template <class T>
__device__ __forceinline__ void load_values(const RecurArgs& a, const void* slab, int64_t i0, const Place& p, float* v)
{
#pragma unroll
    for (int k = 0; k < SEG; k++) v[k] = 0.f;
    load_rows(a, (const T*)slab, a.n, i0, p.c0, p.l, [&](int k, T x) { v[k] = (float)x; });
}

// The map of a segment: forwards h -> gate h + x, or (BACK) from the last step
// to the first into -> gate (into + dh)
template <bool BACK>
__device__ __forceinline__ Map segment_map(const float* gate, const float* v)
{
    Map m{1.f, 0.f};
    bool zero = false;
#pragma unroll
    for (int i = 0; i < SEG; i++) {
        const int k = BACK ? SEG - 1 - i : i;
        m.b = BACK ? advance(gate[k], m.b + v[k], 0.f) : advance(gate[k], m.b, v[k]);
        m.a *= gate[k];
        zero |= gate[k] == 0.f;
    }
    m.a = keep(m.a, zero);
    return m;
}

// Every chunk's map; wave w takes its share of the chunk's segments.  BACK:
// the gradient's, chunks and segments counted from the last.
template <class T, class TG, int NW, bool BACK>
__global__ __launch_bounds__(64 * NW) void maps_kernel(RecurArgs a, Chunks s)
{
    __shared__ float2 box[NW][WAVE];
    const Place p = place<NW, 1>(a.n);
    const Shared g(a.gate_span, p), c(a.cut_span, p);
    const int64_t from = blockIdx.y * s.steps + p.w * (s.steps / NW), segs = (a.T + SEG - 1) / SEG;
    Map m{1.f, 0.f};
    for (int64_t i = from; i < from + s.steps / NW; i += SEG) {
        if (i >= segs * SEG) break;
        const int64_t i0 = BACK ? (segs - 1) * SEG - i : i;
        float gate[SEG], v[SEG];
        load_gates<TG>(a, i0, g, c, gate);
        if (BACK && !a.dh) {
#pragma unroll
            for (int k = 0; k < SEG; k++) v[k] = 0.f;
        } else load_values<T>(a, BACK ? a.dh : a.x, i0, p, v);
        m = compose(m, segment_map<BACK>(gate, v));
    }
    box[p.w][p.lane] = make_float2(m.a, m.b);
    __syncthreads();
    if (p.w != 0) return;
    for (int v = 1; v < NW; v++) m = compose(m, Map{box[v][p.lane].x, box[v][p.lane].y});
    if (p.on) s.maps[blockIdx.y * a.n + p.c()] = make_float2(m.a, m.b);
}

template <class T, class TG, int NW, int CW>
__global__ __launch_bounds__(64 * NW * CW) void recur_kernel(RecurArgs a, Chunks s)
{
    __shared__ float2 box[2][NW][WAVE];
    const Place p = place<NW, CW>(a.n);
    if (NW == 1 && p.c0 >= a.n) return;
    const Shared g(a.gate_span, p), c(a.cut_span, p);
    const int64_t from = blockIdx.y * s.steps, to = from + s.steps < a.T ? from + s.steps : a.T;
    float gate[SEG], x[SEG];
    const auto fetch = [&](int64_t i0) __attribute__((always_inline)) {
        if (i0 >= a.T) return;
        load_gates<TG>(a, i0, g, c, gate);
        load_values<T>(a, a.x, i0, p, x);
    };
    // (the first segment's loads are in flight while the chunks before are composed)
    fetch(from + p.w * SEG);
    float in = reach_chunk<NW>(box[0], s, a.n, p.c(), p.w, p.lane, a.state ? a.state[p.c()] : 0.f);
    int turn = 0;
    for (int64_t i = from; i < to; i += NW * SEG) {
        const int64_t i0 = i + p.w * SEG;
        const bool there = i0 < a.T;
        if (i > from) fetch(i0);
        float h = in;
        if constexpr (NW > 1)
            h = join<NW>(box[turn], p.w, p.lane, there ? segment_map<false>(gate, x) : Map{1.f, 0.f}, in);
        turn ^= 1;
        if (!there) continue;
        if (p.on && a.carry) a.carry[i0 / SEG * a.n + p.c()] = h;
        const int m = i0 + SEG <= a.T ? SEG : (int)(a.T - i0);
        T* row = (T*)a.h + step_at(a, i0) * a.n + p.c0;
        const int64_t next = a.reverse ? -a.n : a.n;
#pragma unroll
        for (int k = 0; k < SEG; k++, row += next) {
            h = advance(gate[k], h, x[k]);
            if (k < m && p.on) row[p.l] = (T)h;
        }
        if constexpr (NW == 1) in = h;
    }
    if (a.last && p.on && p.w == 0 && to == a.T) a.last[p.c()] = in;
}

// The sums over the channels that share a gate, of one segment's products
// d[k] (one a lane): a gate's channels lie side by side, so a wave holds a
// few whole gates and parts of two.  d crosses LDS; then every lane adds the
// channels of (step, gate) pairs, in their order.
template <class TG>
__device__ __forceinline__ void gate_sums(const RecurArgs& a, float (*tile)[WAVE + 1], int64_t i0, const Place& p, const float* d)
{
#pragma unroll
    for (int k = 0; k < SEG; k++) tile[k][p.lane] = p.on ? d[k] : 0.f;
    wave_sync();
    const int64_t first = (uint32_t)p.c0 / a.gate_span, wave = p.c0 / WAVE;
    const int64_t end = p.c0 + WAVE < a.n ? p.c0 + WAVE : a.n;
    const int gates = (int)((uint32_t)(end - 1) / a.gate_span - first) + 1;
    for (int q = p.lane; q < gates * SEG; q += WAVE) {
        const int64_t gate = first + q / SEG;
        const int k = q % SEG;
        if (i0 + k >= a.T) continue;
        const int64_t lo = gate * a.gate_span - p.c0, hi = lo + a.gate_span;
        float sum = 0.f;
        for (int j = lo > 0 ? (int)lo : 0; j < (hi < WAVE ? (int)hi : WAVE); j++) sum += tile[k][j];
        const int64_t at = step_at(a, i0 + k) * a.gates + gate;
        if (a.parts == 1) ((TG*)a.dgate)[at] = (TG)sum;
        else a.part[at * a.parts + (int)(wave - gate * a.gate_span / WAVE)] = sum;
    }
    wave_sync();
}

// The segments from the last to the first: the states before a segment's
// steps again from its carry, the gradient that reaches it as the forward
// pass joins states, then its steps backwards.
template <class T, class TG, int NW, int CW, bool SUMS>
__global__ __launch_bounds__(64 * NW * CW) void recur_backward_kernel(RecurArgs a, Chunks s)
{
    __shared__ float2 box[2][NW][WAVE];
    __shared__ float tiles[SUMS ? NW * CW : 1][SEG][WAVE + 1];
    const Place p = place<NW, CW>(a.n);
    if (NW == 1 && p.c0 >= a.n) return;
    const Shared g(a.gate_span, p), c(a.cut_span, p);
    const int64_t segs = (a.T + SEG - 1) / SEG;
    const int64_t from = blockIdx.y * s.steps, to = from + s.steps < segs * SEG ? from + s.steps : segs * SEG;
    float gate[SEG], before[SEG], dh[SEG];
    uint32_t cut = 0;
    const auto fetch = [&](int64_t i0) __attribute__((always_inline)) {
        if (i0 < 0) return;
        float x[SEG];
        cut = load_gates<TG>(a, i0, g, c, gate);
        load_values<T>(a, a.x, i0, p, x);
        if (a.dh) load_values<T>(a, a.dh, i0, p, dh);
        else {
#pragma unroll
            for (int k = 0; k < SEG; k++) dh[k] = 0.f;
        }
        float h = a.carry[i0 / SEG * a.n + p.c()];
#pragma unroll
        for (int k = 0; k < SEG; k++) {
            before[k] = h;
            h = advance(gate[k], h, x[k]);
        }
    };
    fetch((segs - 1) * SEG - (from + p.w * SEG));
    float in = reach_chunk<NW>(box[0], s, a.n, p.c(), p.w, p.lane, a.dlast ? a.dlast[p.c()] : 0.f);
    int turn = 0;
    for (int64_t i = from; i < to; i += NW * SEG) {
        // counted from the last segment; a wave whose place lies before the first has nothing to do
        const int64_t i0 = (segs - 1) * SEG - (i + p.w * SEG);
        const bool there = i0 >= 0;
        if (i > from) fetch(i0);
        float into = in;
        if constexpr (NW > 1)
            into = join<NW>(box[turn], p.w, p.lane, there ? segment_map<true>(gate, dh) : Map{1.f, 0.f}, in);
        if (there) {
            const int m = i0 + SEG <= a.T ? SEG : (int)(a.T - i0);
            const int64_t next = a.reverse ? -a.n : a.n, at = step_at(a, i0 + SEG - 1) * a.n + p.c0;
            T* row = (T*)a.dx + at;
            TG* gate_row = (TG*)a.dgate + at;
#pragma unroll
            for (int k = SEG - 1; k >= 0; k--, row -= next, gate_row -= next) {
                const float gk = into + dh[k];
                if (k < m && p.on) row[p.l] = (T)gk;
                into = advance(gate[k], gk, 0.f);
                dh[k] = (cut >> k & 1) ? 0.f : gk * before[k];
                if (!SUMS && a.dgate && k < m && p.on) gate_row[p.l] = (TG)dh[k];
            }
            if constexpr (SUMS) gate_sums<TG>(a, tiles[NW == 1 ? (int)threadIdx.x >> 6 : p.w], i0, p, dh);
        }
        if constexpr (NW == 1) in = into;
        turn ^= 1;
    }
    if (a.dstate && p.on && p.w == 0 && to == segs * SEG) a.dstate[p.c()] = in;
}

// ------------------------------------------------------------- pairs of channels
// 16-bit slabs of many channels: a lane takes two neighbouring channels (one
// 4-byte load a step), kept as they lie in memory until their step.  The
// arguments count pairs: n, gate_span and cut_span are halved, a pair shares its
// cut and, where gates are shared (SHARED), its gate.
template <class T>
struct Two { T a, b; };

template <class T, class TG, bool SHARED>
struct PairSegment {
    Two<T> v[SEG];
    TG gate[SHARED ? SEG : 1];
    Two<TG> gates[SHARED ? 1 : SEG];
    uint32_t cut = 0;

    __device__ __forceinline__ void load_gates(const RecurArgs& a, int64_t i0, const Place& p, const Shared& g, const Shared& c)
    {
        cut = 0;
        if constexpr (SHARED) {
            if (a.gate) load_rows(a, (const TG*)a.gate, a.gates, i0, g.first, g.l, [&](int k, TG x) { gate[k] = x; });
        } else {
            load_rows(a, (const Two<TG>*)a.gate, a.n, i0, p.c0, p.l, [&](int k, Two<TG> x) { gates[k] = x; });
        }
        if (a.cut) load_rows(a, a.cut, a.cuts, i0, c.first, c.l, [&](int k, uint8_t x) { cut |= (x ? 1u : 0u) << k; });
    }
    __device__ __forceinline__ float2 at(const RecurArgs& a, int k) const
    {
        float2 r;
        if constexpr (SHARED) r.x = r.y = a.gate ? (float)gate[k] : a.gate_value;
        else r = make_float2((float)gates[k].a, (float)gates[k].b);
        return cut >> k & 1 ? make_float2(0.f, 0.f) : r;
    }
};

template <class T, class TG, bool SHARED>
__global__ __launch_bounds__(256) void recur_pair_kernel(RecurArgs a)
{
    const Place p = place<1, 4>(a.n);
    if (p.c0 >= a.n) return;
    const Shared g(a.gate_span, p), c(a.cut_span, p);
    const int64_t next = a.reverse ? -a.n : a.n;
    float2 h = a.state ? ((const float2*)a.state)[p.c()] : make_float2(0.f, 0.f);
    for (int64_t i0 = 0; i0 < a.T; i0 += SEG) {
        PairSegment<T, TG, SHARED> s;
        s.load_gates(a, i0, p, g, c);
        load_rows(a, (const Two<T>*)a.x, a.n, i0, p.c0, p.l, [&](int k, Two<T> x) { s.v[k] = x; });
        if (p.on && a.carry) ((float2*)a.carry)[i0 / SEG * a.n + p.c()] = h;
        const int m = i0 + SEG <= a.T ? SEG : (int)(a.T - i0);
        Two<T>* row = (Two<T>*)a.h + step_at(a, i0) * a.n + p.c0;
#pragma unroll
        for (int k = 0; k < SEG; k++, row += next) {
            if (k >= m) continue;
            const float2 q = s.at(a, k);
            h.x = advance(q.x, h.x, (float)s.v[k].a);
            h.y = advance(q.y, h.y, (float)s.v[k].b);
            if (p.on) row[p.l] = Two<T>{(T)h.x, (T)h.y};
        }
    }
    if (a.last && p.on) ((float2*)a.last)[p.c()] = h;
}

template <class T, class TG, bool SHARED>
__global__ __launch_bounds__(256) void recur_backward_pair_kernel(RecurArgs a)
{
    __shared__ float tiles[SHARED ? 4 : 1][SEG][WAVE + 1];
    const Place p = place<1, 4>(a.n);
    if (p.c0 >= a.n) return;
    const Shared g(a.gate_span, p), c(a.cut_span, p);
    const int64_t next = a.reverse ? -a.n : a.n;
    float2 into = a.dlast ? ((const float2*)a.dlast)[p.c()] : make_float2(0.f, 0.f);
    for (int64_t i0 = (a.T + SEG - 1) / SEG * SEG - SEG; i0 >= 0; i0 -= SEG) {
        PairSegment<T, TG, SHARED> s;
        Two<T> dh[SEG];
        s.load_gates(a, i0, p, g, c);
        load_rows(a, (const Two<T>*)a.x, a.n, i0, p.c0, p.l, [&](int k, Two<T> x) { s.v[k] = x; });
        if (a.dh) load_rows(a, (const Two<T>*)a.dh, a.n, i0, p.c0, p.l, [&](int k, Two<T> x) { dh[k] = x; });
        const int m = i0 + SEG <= a.T ? SEG : (int)(a.T - i0);
        float2 before[SEG], h = ((const float2*)a.carry)[i0 / SEG * a.n + p.c()];
#pragma unroll
        for (int k = 0; k < SEG; k++) {
            before[k] = h;
            if (k >= m) continue;
            const float2 q = s.at(a, k);
            h.x = advance(q.x, h.x, (float)s.v[k].a);
            h.y = advance(q.y, h.y, (float)s.v[k].b);
        }
        const int64_t at = step_at(a, i0 + SEG - 1) * a.n + p.c0;
        Two<T>* row = (Two<T>*)a.dx + at;
        Two<TG>* gate_row = (Two<TG>*)a.dgate + at;
        float d[SHARED ? SEG : 1];
#pragma unroll
        for (int k = SEG - 1; k >= 0; k--, row -= next, gate_row -= next) {
            if constexpr (SHARED) d[k] = 0.f;
            if (k >= m) continue;
            const float2 q = s.at(a, k);
            const float gx = into.x + (a.dh ? (float)dh[k].a : 0.f), gy = into.y + (a.dh ? (float)dh[k].b : 0.f);
            if (p.on) row[p.l] = Two<T>{(T)gx, (T)gy};
            into.x = advance(q.x, gx, 0.f);
            into.y = advance(q.y, gy, 0.f);
            const bool cut = s.cut >> k & 1;
            const float dx = cut ? 0.f : gx * before[k].x, dy = cut ? 0.f : gy * before[k].y;
            if constexpr (SHARED) d[k] = dx + dy;
            else if (a.dgate && p.on) gate_row[p.l] = Two<TG>{(TG)dx, (TG)dy};
        }
        if constexpr (SHARED) {
            if (a.dgate) gate_sums<TG>(a, tiles[threadIdx.x >> 6], i0, p, d);
        }
    }
    if (a.dstate && p.on) ((float2*)a.dstate)[p.c()] = into;
}

// the waves' parts of every shared gate's sum, in their order
template <class TG>
__global__ __launch_bounds__(256) void gate_parts_kernel(RecurArgs a)
{
    const int64_t gates = a.gates;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.T * gates; i += (int64_t)gridDim.x * 256) {
        const int64_t lo = i % gates * a.gate_span;
        const int pieces = (int)((lo + a.gate_span - 1) / WAVE - lo / WAVE) + 1;
        float s = 0.f;
        for (int p = 0; p < pieces; p++) s += a.part[i * a.parts + p];
        ((TG*)a.dgate)[i] = (TG)s;
    }
}

// (a launch has fewer than 2^32 threads: beyond 2^30 gates they take several)
unsigned gate_parts_blocks(const RecurArgs& a)
{
    const int64_t need = (a.T * a.gates + 255) / 256;
    return (unsigned)(need < (1 << 22) ? need : 1 << 22);
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

// One segment of a lane's steps: for each step the map carry -> gate carry +
// delta, the value (0 where the lane did not act) and whether it acted.
template <class TR, class TV>
__device__ __forceinline__ uint32_t load_steps(const AdvArgs& a, int64_t n, int64_t i0, const Place& p, const Shared& env,
                                      bool acts, float* gate, float* delta, float* value)
{
    uint8_t done[SEG + 1], mark[SEG + 1];       // [k]: of the step before step k
    float next[SEG + 1];
#pragma unroll
    for (int k = 0; k <= SEG; k++) {
        const int64_t t = i0 + k <= a.T ? i0 + k : a.T, b = t > 0 ? t - 1 : 0;
        done[k] = (a.done + b * n + p.c0)[p.l];
        mark[k] = (a.marks + b * a.E + env.first)[env.l];
        next[k] = (float)((const TV*)a.value + t * n + p.c0)[p.l];
    }
#pragma unroll
    for (int k = 0; k < SEG; k++)
        delta[k] = (float)((const TR*)a.reward + (i0 + k < a.T ? i0 + k : a.T - 1) * n + p.c0)[p.l];
    const bool live = i0 > 0 || (a.live + p.c0)[p.l];
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < SEG; k++) {
        const uint8_t m = mark[k + 1];
        const bool before = i0 + k == 0 ? live : (mark[k] & GW_MARK_END) || !done[k];
        const bool ok = acts && before && !(m & (GW_MARK_RESET | GW_MARK_SKIP)) && i0 + k < a.T;
        const bool final = done[k + 1] || (m & GW_MARK_END);
        const float d = delta[k] - next[k] + (final ? 0.f : a.gamma * next[k + 1]);
        delta[k] = ok ? d : 0.f;
        value[k] = ok ? next[k] : 0.f;
        gate[k] = i0 + k >= a.T ? 1.f : ok && !final && !(m & GW_MARK_TRUNCATED) ? a.gamma * a.lam : 0.f;
        bits |= (ok ? 1u : 0u) << k;
    }
    return bits;
}

// The recurrence from the last step to the first, split as the gradient's
// (MAPS: the chunks' maps only).  Memory bounds it: 100 steps of 4096 envs of 64
// lanes, float64 rewards and float32 values: 127 us, 578 MB at 4.6 TB/s (a copy:
// 5.2).  5003 steps of 15 lanes: 7.8 us of maps and 12 us of walk, both latency.
template <class TR, class TV, int NW, int CW, bool MAPS>
__global__ __launch_bounds__(64 * NW * CW) void advantages_kernel(AdvArgs a, Chunks s)
{
    __shared__ float2 box[2][NW][WAVE];
    const int64_t n = a.E * a.A;
    const Place p = place<NW, CW>(n);
    if (NW == 1 && p.c0 >= n) return;
    const Shared env((uint32_t)a.A, p);
    const bool acts = !a.acts || a.acts[(uint32_t)p.c() % (uint32_t)a.A];
    const int64_t segs = (a.T + SEG - 1) / SEG;
    const int64_t from = blockIdx.y * s.steps, to = from + s.steps < segs * SEG ? from + s.steps : segs * SEG;
    float in = 0.f;
    Map whole{1.f, 0.f};
    if (!MAPS) in = reach_chunk<NW>(box[0], s, n, p.c(), p.w, p.lane, 0.f);
    int turn = 0;
    for (int64_t i = from; i < to; i += NW * SEG) {
        const int64_t i0 = (segs - 1) * SEG - (i + p.w * SEG);
        const bool there = i0 >= 0;
        float gate[SEG], delta[SEG], value[SEG];
        uint32_t ok = 0;
        Map m{1.f, 0.f};
        if (there) {
            ok = load_steps<TR, TV>(a, n, i0, p, env, acts, gate, delta, value);
            bool zero = false;
#pragma unroll
            for (int k = SEG - 1; k >= 0; k--) {
                m.b = advance(gate[k], m.b, delta[k]);
                m.a *= gate[k];
                zero |= gate[k] == 0.f;
            }
            m.a = keep(m.a, zero);
        }
        float h = in;
        if constexpr (MAPS) {
            box[turn][p.w][p.lane] = make_float2(m.a, m.b);
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NW; v++) whole = compose(whole, Map{box[turn][v][p.lane].x, box[turn][v][p.lane].y});
        } else if (NW > 1) {
            h = join<NW>(box[turn], p.w, p.lane, m, in);
        }
        if (!MAPS && there) {
#pragma unroll
            for (int k = SEG - 1; k >= 0; k--) {
                h = advance(gate[k], h, delta[k]);
                if (p.on && i0 + k < a.T) {
                    const int64_t row = (i0 + k) * n + p.c0;
                    const bool acted = ok >> k & 1;
                    (a.advantage + row)[p.l] = h;
                    (a.target + row)[p.l] = acted ? h + value[k] : 0.f;
                    (a.valid + row)[p.l] = acted;
                }
            }
        }
        if (NW == 1) in = h;
        turn ^= 1;
    }
    if (MAPS && p.w == 0 && p.on) s.maps[blockIdx.y * n + p.c()] = make_float2(whole.a, whole.b);
}

// parts of a shared gate's sum: the waves that its channels can lie in
int64_t gate_pieces(int64_t gate_span) { return WAVE % gate_span == 0 ? 1 : (gate_span - 1) / WAVE + 2; }

// How the steps are split.  A wave keeps 2 SEG values a lane in flight; FILL
// waves keep the memory busy (256 CUs, 16 each), and chunks are made for twice
// as many: 65537 steps of 96 channels, forward and backward, took 84 us with
// FILL, 71 with 2 FILL, 87 with 4 FILL waves of chunks (more maps to compose).
constexpr int64_t FILL = 4096;
struct Split { int nw; Chunks s; };

Split split_steps(int64_t T, int64_t n, float2* maps)
{
    const int64_t waves = (n + WAVE - 1) / WAVE, segs = (T + SEG - 1) / SEG;
    Split r{};
    r.nw = waves >= FILL || segs <= 1 ? 1 : waves * 4 >= FILL || segs <= 4 ? 4 : 8;
    const int64_t tile = (int64_t)r.nw * SEG, tiles = (T + tile - 1) / tile;
    int64_t chunks = r.nw == 8 ? 2 * FILL / (waves * r.nw) : 1;
    chunks = chunks < 1 ? 1 : chunks > tiles ? tiles : chunks;
    if (chunks <= 2) chunks = 1;                        // two launches do not pay for so few
    const int64_t per = chunks > 1 ? (tiles + chunks - 1) / chunks : (tiles > 0 ? tiles : 1);
    r.s.count = chunks > 1 ? (int32_t)((tiles + per - 1) / per) : 1;
    r.s.steps = per * tile;
    r.s.maps = maps;
    return r;
}

template <class TR, class TV>
void launch_advantages(const AdvArgs& a, void* workspace, hipStream_t st)
{
    const int64_t n = a.E * a.A, waves = (n + WAVE - 1) / WAVE;
    const Split q = split_steps(a.T, n, (float2*)workspace);
    const dim3 grid((unsigned)waves, q.s.count);
    if (q.s.count > 1) hipLaunchKernelGGL((advantages_kernel<TR, TV, 8, 1, true>), grid, dim3(512), 0, st, a, q.s);
    if (q.nw == 1)
        hipLaunchKernelGGL((advantages_kernel<TR, TV, 1, 4, false>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, q.s);
    else if (q.nw == 4) hipLaunchKernelGGL((advantages_kernel<TR, TV, 4, 1, false>), grid, dim3(256), 0, st, a, q.s);
    else hipLaunchKernelGGL((advantages_kernel<TR, TV, 8, 1, false>), grid, dim3(512), 0, st, a, q.s);
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Whether 16-bit channels go in pairs: where channels alone fill the device
// (20 steps of 1048576 channels bf16, forward and backward: 89 us, 135 us one
// a lane), pairs share what is shared and nothing lies at odd places.
template <class T, class TG>
bool take_pairs(const RecurArgs& a, RecurArgs* b)
{
    if (sizeof(T) != 2 || a.n % 2 || split_steps(a.T, a.n, nullptr).nw != 1 || a.n / WAVE / 2 < FILL) return false;
    const bool shared = !a.gate || a.gate_span > 1;
    if ((shared && a.gate && a.gate_span % 2) || (a.cut && a.cut_span % 2)) return false;
    if (!aligned(a.x, 4) || !aligned(a.h, 4) || !aligned(a.dh, 4) || !aligned(a.dx, 4)) return false;
    if (!shared && (!aligned(a.gate, 2 * sizeof(TG)) || !aligned(a.dgate, 2 * sizeof(TG)))) return false;
    if (!aligned(a.state, 8) || !aligned(a.last, 8) || !aligned(a.carry, 8) || !aligned(a.dlast, 8) || !aligned(a.dstate, 8))
        return false;
    *b = a;
    b->n = a.n / 2;
    b->gate_span = shared && a.gate ? a.gate_span / 2 : 1;
    b->cut_span = a.cut ? a.cut_span / 2 : 1;
    b->gates = b->n / b->gate_span;
    b->cuts = b->n / b->cut_span;
    b->parts = (int32_t)gate_pieces(b->gate_span);
    return true;
}

template <class T, class TG>
void launch_recurrence(const RecurArgs& a, void* workspace, hipStream_t st)
{
    RecurArgs b;
    if constexpr (sizeof(T) == 2) if (take_pairs<T, TG>(a, &b)) {
        const dim3 blocks((unsigned)((b.n + 4 * WAVE - 1) / (4 * WAVE)));
        if (!a.gate || a.gate_span > 1) hipLaunchKernelGGL((recur_pair_kernel<T, TG, true>), blocks, dim3(256), 0, st, b);
        else hipLaunchKernelGGL((recur_pair_kernel<T, TG, false>), blocks, dim3(256), 0, st, b);
        return;
    }
    const Split q = split_steps(a.T, a.n, (float2*)workspace);
    const int64_t waves = (a.n + WAVE - 1) / WAVE;
    const dim3 grid((unsigned)waves, q.s.count);
    if (q.s.count > 1) hipLaunchKernelGGL((maps_kernel<T, TG, 8, false>), grid, dim3(512), 0, st, a, q.s);
    if (q.nw == 1) hipLaunchKernelGGL((recur_kernel<T, TG, 1, 4>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, q.s);
    else if (q.nw == 4) hipLaunchKernelGGL((recur_kernel<T, TG, 4, 1>), grid, dim3(256), 0, st, a, q.s);
    else hipLaunchKernelGGL((recur_kernel<T, TG, 8, 1>), grid, dim3(512), 0, st, a, q.s);
}

template <class T, class TG, bool SUMS>
void launch_backward(const RecurArgs& a, void* workspace, hipStream_t st)
{
    const Split q = split_steps(a.T, a.n, (float2*)workspace);
    const int64_t waves = (a.n + WAVE - 1) / WAVE;
    const dim3 grid((unsigned)waves, q.s.count);
    if (q.s.count > 1) hipLaunchKernelGGL((maps_kernel<T, TG, 8, true>), grid, dim3(512), 0, st, a, q.s);
    if (q.nw == 1)
        hipLaunchKernelGGL((recur_backward_kernel<T, TG, 1, 4, SUMS>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, q.s);
    else if (q.nw == 4) hipLaunchKernelGGL((recur_backward_kernel<T, TG, 4, 1, SUMS>), grid, dim3(256), 0, st, a, q.s);
    else hipLaunchKernelGGL((recur_backward_kernel<T, TG, 8, 1, SUMS>), grid, dim3(512), 0, st, a, q.s);
    if (SUMS && a.parts > 1)
        hipLaunchKernelGGL((gate_parts_kernel<TG>), dim3(gate_parts_blocks(a)), dim3(256), 0,
                           st, a);
}

template <class T, class TG>
void launch_backward(const RecurArgs& a, void* workspace, hipStream_t st)
{
    RecurArgs b;
    if constexpr (sizeof(T) == 2) if (take_pairs<T, TG>(a, &b)) {
        const dim3 blocks((unsigned)((b.n + 4 * WAVE - 1) / (4 * WAVE)));
        if (!a.gate || a.gate_span > 1) hipLaunchKernelGGL((recur_backward_pair_kernel<T, TG, true>), blocks, dim3(256), 0, st, b);
        else hipLaunchKernelGGL((recur_backward_pair_kernel<T, TG, false>), blocks, dim3(256), 0, st, b);
        if (b.dgate && a.gate_span > 1 && b.parts > 1)
            hipLaunchKernelGGL((gate_parts_kernel<TG>), dim3(gate_parts_blocks(b)), dim3(256), 0, st, b);
        return;
    }
    if (a.dgate && a.gate_span > 1) launch_backward<T, TG, true>(a, workspace, st);
    else launch_backward<T, TG, false>(a, workspace, st);
}

gw_status check_recurrence(int32_t dtype, int32_t gate_dtype, int64_t T, int64_t n, const void* x, const void* gate,
                           int64_t gate_span, float gate_value, const uint8_t* cut, int64_t cut_span)
{
    LEARN_NEED(dtype >= GW_T_F32 && dtype <= GW_T_BF16, "unknown dtype %d", dtype);
    LEARN_NEED(gate_dtype == dtype || gate_dtype == GW_T_F32, "gate_dtype %d with dtype %d: the same or GW_T_F32",
               gate_dtype, dtype);
    LEARN_NEED(T >= 0 && n >= 0 && T <= (INT64_C(1) << 31) && n < (INT64_C(1) << 31), "%lld steps of %lld channels",
               (long long)T, (long long)n);
    LEARN_NEED(T == 0 || n == 0 || x, "x: null pointer");
    LEARN_NEED(gate_span >= 1 && n % gate_span == 0, "gate_span %lld for %lld channels", (long long)gate_span, (long long)n);
    LEARN_NEED(gate || isfinite(gate_value), "gate_value is not finite");
    LEARN_NEED(!cut || (cut_span >= 1 && n % cut_span == 0), "cut_span %lld for %lld channels", (long long)cut_span,
               (long long)n);
    return GW_OK;
}

int64_t maps_bytes(int64_t T, int64_t n)
{
    const Split q = split_steps(T, n, nullptr);
    return q.s.count > 1 ? q.s.count * n * (int64_t)sizeof(float2) : 0;
}

}  // namespace

extern "C" {

int64_t gw_recurrence_workspace(int64_t n_steps, int64_t n) { return n_steps <= 0 || n <= 0 ? 0 : maps_bytes(n_steps, n); }

gw_status gw_recurrence(int32_t dtype, int32_t gate_dtype, int64_t n_steps, int64_t n,
                        const void* x, const void* gate, int64_t gate_span, float gate_value,
                        const uint8_t* cut, int64_t cut_span, const float* state, int32_t reverse,
                        void* h, float* last, float* carry,
                        void* workspace, int64_t workspace_bytes, void* stream)
{
    const gw_status s = check_recurrence(dtype, gate_dtype, n_steps, n, x, gate, gate_span, gate_value, cut, cut_span);
    if (s != GW_OK) return s;
    LEARN_NEED(n_steps == 0 || n == 0 || h, "h: null pointer");
    const int64_t need = gw_recurrence_workspace(n_steps, n);
    LEARN_NEED(need == 0 || (workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need),
               "workspace: %lld bytes, 8-byte aligned, are needed", (long long)need);
    if (n == 0) return GW_OK;
    RecurArgs a{};
    a.T = n_steps; a.n = n; a.x = x; a.gate = gate; a.gate_span = (uint32_t)gate_span; a.gate_value = gate_value;
    a.cut = cut; a.cut_span = cut ? (uint32_t)cut_span : 1; a.gates = n / gate_span; a.cuts = n / a.cut_span;
    a.state = state; a.reverse = reverse;
    a.h = h; a.last = last; a.carry = carry;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GW_T_F32) launch_recurrence<float, float>(a, workspace, st);
    else if (dtype == GW_T_F16) gate_dtype == dtype ? launch_recurrence<f16, f16>(a, workspace, st) : launch_recurrence<f16, float>(a, workspace, st);
    else gate_dtype == dtype ? launch_recurrence<bf16, bf16>(a, workspace, st) : launch_recurrence<bf16, float>(a, workspace, st);
    LEARN_LAUNCHED();
    return GW_OK;
}

int64_t gw_recurrence_backward_workspace(int64_t n_steps, int64_t n, int64_t gate_span)
{
    if (n_steps <= 0 || n <= 0 || gate_span < 1) return 0;
    const int64_t pieces = gate_span > 1 ? gate_pieces(gate_span) : 1;
    return maps_bytes(n_steps, n) + (pieces > 1 ? n_steps * (n / gate_span) * pieces * 4 : 0);
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
    const int64_t need = gw_recurrence_backward_workspace(n_steps, n, gate_span);
    LEARN_NEED(need == 0 || (workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need),
               "workspace: %lld bytes, 8-byte aligned, are needed", (long long)need);
    if (n == 0) return GW_OK;
    RecurArgs a{};
    a.T = n_steps; a.n = n; a.x = x; a.gate = gate; a.gate_span = (uint32_t)gate_span; a.gate_value = gate_value;
    a.cut = cut; a.cut_span = cut ? (uint32_t)cut_span : 1; a.gates = n / gate_span; a.cuts = n / a.cut_span;
    a.reverse = reverse; a.carry = const_cast<float*>(carry);
    a.dh = dh; a.dlast = dlast; a.dx = dx; a.dgate = dgate; a.dstate = dstate;
    a.part = (float*)((char*)workspace + maps_bytes(n_steps, n)); a.parts = (int32_t)gate_pieces(gate_span);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GW_T_F32) launch_backward<float, float>(a, workspace, st);
    else if (dtype == GW_T_F16) gate_dtype == dtype ? launch_backward<f16, f16>(a, workspace, st) : launch_backward<f16, float>(a, workspace, st);
    else gate_dtype == dtype ? launch_backward<bf16, bf16>(a, workspace, st) : launch_backward<bf16, float>(a, workspace, st);
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
    LEARN_NEED(dtype >= GW_T_F32 && dtype <= GW_T_BF16, "unknown dtype %d", dtype);
    LEARN_NEED(n_steps >= 0 && n_envs >= 0 && n_lanes >= 1 && n_lanes < (INT64_C(1) << 31) &&
                   n_envs <= ((INT64_C(1) << 31) - 1) / n_lanes,
               "%lld steps of %lld envs of %lld lanes", (long long)n_steps, (long long)n_envs, (long long)n_lanes);
    LEARN_NEED(isfinite(gamma) && isfinite(lam), "gamma or lam is not finite");
    if (n_steps == 0 || n_envs == 0) return GW_OK;
    LEARN_NEED(reward && value && done && marks && live && advantage && target && valid, "null pointer");
    const AdvArgs a{n_steps, n_envs, n_lanes, reward, value, done, marks, live, acts, gamma, lam, advantage, target, valid};
    const int64_t need = gw_recurrence_workspace(n_steps, n_envs * n_lanes);
    LEARN_NEED(need == 0 || (workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need),
               "workspace: %lld bytes, 8-byte aligned, are needed", (long long)need);
    const hipStream_t st = (hipStream_t)stream;
    if (reward_f64) {
        if (dtype == GW_T_F32) launch_advantages<double, float>(a, workspace, st);
        else if (dtype == GW_T_F16) launch_advantages<double, f16>(a, workspace, st);
        else launch_advantages<double, bf16>(a, workspace, st);
    } else {
        if (dtype == GW_T_F32) launch_advantages<float, float>(a, workspace, st);
        else if (dtype == GW_T_F16) launch_advantages<float, f16>(a, workspace, st);
        else launch_advantages<float, bf16>(a, workspace, st);
    }
    LEARN_LAUNCHED();
    return GW_OK;
}

}  // extern "C"
