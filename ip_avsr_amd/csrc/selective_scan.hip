// Selective state-space scan over a (B, T, D) tensor: every channel d drives N states with its own decays, a step size per frame and
// input / output rows B_t, C_t shared by the channels of a group; forward, backward and the form for single frames.
//
//   dt = softplus(delta + delta_bias)  (or delta + delta_bias)
//   a = exp(dt A[d, n]),  h[t, d, n] = a h[t-1, d, n] + dt u B[t, n],  y = sum_n h C[t, n] + D[d] u,  y *= z sigmoid(z) where gated
//   back: dh[t] = dy C[t] + a[t+1] dh[t+1],  e = a h[t-1]
//     ddt = sum_n dh A e + u sum_n dh B,  du = dt sum_n dh B + D dy,  dA = sum dh dt e,  dB = sum_d dh dt u,  dC = sum_d dy h
//
// Bound: the vector pipe.  A (t, d, n) costs a multiply, an exp2 (a quarter of the rate), a multiply and two fused multiply-adds
// forward -- 8 issue slots of a plain instruction -- and about 17 backward, against 8 / N bytes of bfloat16 traffic.
//
// Layout: a quad of lanes owns NC channels and splits their states, lane `ng` of it NS of them, so a lane keeps NC NS = 4 states and
// decays in registers (8 where N > 16) and B_t, C_t cost it NS values each (staged through LDS as float32, once for the workgroup).
// What belongs to a (frame, channel) and not to a state -- the step size, the gate, all loads and stores -- is done once: the quad
// covers 4 / NC frames x NC channels, one per lane, and hands dt and dt u round by quad_perm; a sum over the states is a transposing
// reduction of 4 values over the quad (9 instructions) that leaves each lane the one it owns.  A workgroup is 4 waves of 16 NC
// channels.  More states per lane would save a tenth of the instructions and cost the registers that the backward pass needs.
//
// Frames go by segments of 8 (4 where N > 16 or N <= 4), the loads of the next ones in flight; a segment has no branch in it.  The backward
// pass walks them from the end: from the state the forward pass kept at the segment's start it recomputes a and e of the segment into
// registers, then runs the adjoint.  dB and dC are summed over the lanes of a wave by exchanging halves (permlane swaps, row
// rotations), over the workgroup's waves in LDS and over workgroups by a second launch; dA, dD and the bias' gradient stay in registers
// over all frames of a workgroup's utterances.  All sums run in a fixed order.
// 8 x 2048 x 2048 x 16 bfloat16, gated: forward 285 us with what training keeps, 0.53 us per 10^6 (t, d, n) where the 8 slots take 0.20
// (1024 waves, one per SIMD, the pipe 47 % busy: nothing covers a wave's own waits; with four per SIMD 0.33), backward 469 us (26 vector
// instructions a (t, d, n), the pipe 90 % busy) behind 131 us for the pieces alone.
// Frames at and behind lens[b] are padding: not read, zero in y and the frame gradients; the state passes them unchanged.
#include "seq_common.h"
#include <type_traits>

namespace adn {
namespace seq {

namespace {

constexpr int kMaxStates = 32;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f;

struct ScanParams {
    const int32_t* lens;
    const float* A;                   // [D][N]
    const float* Dp;                  // [D] or null
    const float* dbias;               // [D] or null
    const float* state_in;            // [B][D][N] or null (zeros)
    float* state_out;                 // [B][D][N]
    float* ckpt;                      // states before every segment: [B][nseg][ctiles][P / 4][64][4], or null
    const float* dlast;               // backward: gradient of state_out, or null
    float* dstate;                    // backward: gradient of state_in, or null
    float* part_bc;                   // backward: [bpg][B][nseg][G][SEG][2][4 NS]
    float* part_a;                    // backward: [nbg][chunks][ctiles][64 P + 2 * 16 NC]
    int B, T, D, N, G, Dg;            // Dg = D / G channels per group
    int nseg, bpg, ctiles;            // segments; workgroups per group; waves of all workgroups along the channels
    int nbg, per_bg;                  // backward: groups of utterances, utterances per group
    int chunks, spc;                  // pieces that the time axis is split into, segments of a piece
    float* local;                     // chunks > 1: what a piece alone leaves, [B][chunks][ctiles][P / 4][64][4] ...
    float* dsum;                      // ... and its sum of dt, [B][chunks][ctiles][16 NC]
    int softplus;
};

// channels of a quad and frames of a segment: 4 (channel, state) pairs per lane and 8 frames; 8 pairs and 4 frames where N > 16, which
// keeps what a segment takes in registers, and 4 frames where N <= 4, whose lanes own a frame of every channel and would spill the rest
// (32 x 512 x 2048 x 4: backward 228 us, with 8 frames 273; of 8 states 8 frames 303 us, 4 frames 344)
constexpr int channels_per_quad(int ns) { return ns == 8 ? 1 : 4 / ns; }
constexpr int segment_frames(int ns) { return ns == 1 || ns == 8 ? 4 : 8; }

// log(1 + exp(x)), relative accuracy also where it is small: log1p(e) = 2 atanh(e / (2 + e)) of e = exp(-|x|) <= 1, whose odd series
// in s = e / (2 + e) <= 1/3 is cut where the rest is below 2^-26 of it
__device__ __forceinline__ float softplusf(float x) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float r = 1.f / 15.f;
    r = fmaf(r, q, 1.f / 13.f);
    r = fmaf(r, q, 1.f / 11.f);
    r = fmaf(r, q, 1.f / 9.f);
    r = fmaf(r, q, 1.f / 7.f);
    r = fmaf(r, q, 1.f / 5.f);
    r = fmaf(r, q, 1.f / 3.f);
    r = fmaf(r, q, 1.f);
    return fmaxf(x, 0.f) + 2.f * s * r;
}

// A as the exponent's factor for base 2.  The product passes float32's range from |A| = 2.36e38 on (the lowest value is what a state that
// keeps nothing has), and an infinity times a step size of 0, or times a gradient of 0, would be NaN: the largest number has the same decays
// (and the derivative by a step size of 0 is that of 2.36e38)
__device__ __forceinline__ float decay2(float A) {
    const float v = A * kLog2e;
    return __builtin_isinf(v) ? __builtin_copysignf(3.40282347e38f, v) : v;
}

__device__ __forceinline__ float bcast(float v, int q) {
    switch (q) {
        case 0: return quad_bcast<0>(v);
        case 1: return quad_bcast<1>(v);
        case 2: return quad_bcast<2>(v);
        default: return quad_bcast<3>(v);
    }
}
// lane ng of a quad: the sum over the quad of v[ng]
__device__ __forceinline__ float quad_gather(const float (&v)[4], bool b0, bool b1) {
    const float x0 = (b0 ? v[1] : v[0]) + dpp<kQuadXor1>(b0 ? v[0] : v[1]);
    const float x1 = (b0 ? v[3] : v[2]) + dpp<kQuadXor1>(b0 ? v[2] : v[3]);
    return (b1 ? x1 : x0) + dpp<kQuadXor2>(b1 ? x0 : x1);
}

// where a wave and its lanes stand
template <int NS> struct Place {
    static constexpr int NC = channels_per_quad(NS), SEG = segment_frames(NS), TQ = 4 / NC, WC = 16 * NC, P = NC * NS, Q = SEG / TQ;
    static constexpr int STAGE = SEG * 8 * NS, SPT = (STAGE + 255) / 256;      // values of B and C in a segment, and per thread
    int lane, wv, ng, cl, g, ctile, c0, cend, oc, otp;
    bool ocv, b0, b1;
    int st_s, st_at, st_which;        // the staged value of this thread: frame (none: far behind any), place in the row of its group, B or C
    __device__ __forceinline__ Place(const ScanParams& p, int cblk) {
        lane = threadIdx.x & 63;
        wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
        ng = lane & 3;
        cl = lane >> 2;
        g = cblk / p.bpg;
        const int tg = (cblk - g * p.bpg) * 4 + wv;
        ctile = cblk * 4 + wv;
        c0 = g * p.Dg + tg * WC + cl * NC;          // the quad's first channel
        cend = (g + 1) * p.Dg;
        oc = c0 + ng % NC;                          // the channel and, below, the frame of the quad that this lane owns
        otp = ng / NC;
        ocv = oc < cend;
        b0 = ng & 1;
        b1 = ng >> 1;
        st_s = (int)threadIdx.x / (8 * NS);
        st_which = ((int)threadIdx.x / (4 * NS)) & 1;
        const int n = (int)threadIdx.x % (4 * NS);
        st_at = g * p.N + n;
        if ((int)threadIdx.x >= STAGE || n >= p.N) st_s = 1 << 30;
    }
};
static_assert(Place<1>::SPT == 1 && Place<2>::SPT == 1 && Place<4>::SPT == 1 && Place<8>::SPT == 1, "one staged value per thread");

// a (B, T, D) tensor as a wave walks one utterance: buffer accesses from a uniform base at a segment's first frame, with a 32-bit offset
// per lane (check() holds the frame stride below 2^26).  A lane without a channel, or without a frame, gets the offset that the bounds
// check turns away: its load is 0, its store is dropped, and no branch stands between the loads in flight
constexpr uint32_t kNowhere = 0x80000000u;
template <typename T> struct Walk {
    char* p;                           // the segment's first frame
    uint32_t frame;                    // bytes between frames
    uint32_t off;                      // of the lane's first frame in a segment
    __device__ __forceinline__ Walk(const View<T>& v, int b, int t0, int frame_of_lane, int c, bool on)
        : p(reinterpret_cast<char*>(const_cast<std::remove_const_t<T>*>(v.p + b * v.sb + t0 * v.st))), frame((uint32_t)v.st * (uint32_t)sizeof(T)),
          off(on ? (uint32_t)frame_of_lane * frame + (uint32_t)c * (uint32_t)sizeof(T) : kNowhere) {}
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t base() const { return __builtin_amdgcn_make_buffer_rsrc(p, 0, 0x7FFFFFFF, 0x00027000); }
    // ... where the walk stays at its start: the backward pass holds seven of them and has no scalar registers to move them in
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t base(int t0) const {
        return __builtin_amdgcn_make_buffer_rsrc(p + (uint64_t)(uint32_t)t0 * frame, 0, 0x7FFFFFFF, 0x00027000);
    }
    // on by FRAMES; a place outside the tensor is harmless as long as every lane is turned away there
    template <int FRAMES> __device__ __forceinline__ void move() { p += (int64_t)FRAMES * (int64_t)frame; }
    // `ahead` frames behind the lane's first; `on`: whether there is such a frame
    __device__ __forceinline__ uint32_t at(int ahead, bool on) const { return on ? off + (uint32_t)ahead * frame : kNowhere; }
};
__device__ __forceinline__ float raw_to_float(uint32_t v, float) { return __builtin_bit_cast(float, v); }
__device__ __forceinline__ float raw_to_float(uint32_t v, __bf16) { return __builtin_bit_cast(float, v << 16); }
// the bits of an element (a bfloat16 in the lower half)
template <typename T> __device__ __forceinline__ uint32_t buf_load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (sizeof(T) == 2) return (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
}
template <typename T> __device__ __forceinline__ void buf_store(__amdgpu_buffer_rsrc_t r, uint32_t off, float v) {
    if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (T)v), r, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), r, off, 0, 0);
}

// LDS reads stay on their side of this point: a frame's B and C are read while the frame before is computed.  Without it the compiler
// puts each read right before its use, and a lone wave on its SIMD waits for every one
__device__ __forceinline__ void hold_reads() { __builtin_amdgcn_sched_barrier(0x277); }

template <int P> __device__ __forceinline__ int64_t ckpt_at(const ScanParams& p, int b, int seg, int ctile) {
    return (((int64_t)b * p.nseg + seg) * p.ctiles + ctile) * 64 * P;
}

template <int P> __device__ __forceinline__ int64_t local_at(const ScanParams& p, int b, int chunk, int ctile) {
    return (((int64_t)b * p.chunks + chunk) * p.ctiles + ctile) * 64 * P;
}
// x (a state, or a state's gradient) carried over a piece: x = what the piece alone leaves + exp(A sum dt) x.  The factor may be no float32
// number where the product is -- the state shrinks from a large one, or grows from a tiny one -- so it is applied in halves: down to
// 2^-252 and up to 2^256.  CAREFUL: in thirds of at most 2^127, for what a growth past that makes of a state of zero (NaN in halves)
// or of a denormal one
template <int NS, bool CAREFUL>
__device__ __forceinline__ void carry_over(const ScanParams& p, const Place<NS>& l, int b, int chunk, const float (&A2)[Place<NS>::NC][NS],
                                           float (&x)[Place<NS>::NC][NS]) {
    constexpr int P = Place<NS>::P, NC = Place<NS>::NC, WC = Place<NS>::WC;
    const float* src = p.local + local_at<P>(p, b, chunk, l.ctile) + l.lane * 4;
    const float* ds = p.dsum + (((int64_t)b * p.chunks + chunk) * p.ctiles + l.ctile) * WC + l.cl * NC;
    float v[P], d[NC];
#pragma unroll
    for (int m = 0; m < P / 4; ++m) load_vec<float, 4>(src + m * 256, v + m * 4);
    load_vec<float, NC>(ds, d);
#pragma unroll
    for (int k = 0; k < NC; ++k) d[k] *= CAREFUL ? 1.f / 3.f : 0.5f;
#pragma unroll
    for (int m = 0; m < P; ++m) {
        float& s = x[m / NS][m % NS];
        const float e = d[m / NS] * A2[m / NS][m % NS], f = __builtin_amdgcn_exp2f(CAREFUL ? fminf(e, 127.f) : e);
        s = fmaf(CAREFUL ? s * f * f : s * f, f, v[m]);
    }
}
template <int NC, int NS> __device__ __forceinline__ bool all_finite(const float (&x)[NC][NS]) {
    bool on = true;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j) on = on && __builtin_isfinite(x[k][j]);
    return on;
}

// The states (gradients) of a lane over the frames from .. to themselves, for where they do not come out finite over the pieces: a piece
// alone can overflow that frame by frame would not, where its input cancels what an earlier state grows to.  States that are all NaN
// end it: nothing changes them.  Backward (in: dy, m: C, z: the gate or null) from the end.
template <typename T, int NS, bool BACK>
__device__ __forceinline__ void over_frames(const View<const T>& in, const View<const T>& delta, const View<const T>& m, const View<const T>& z, const ScanParams& p,
                                            const Place<NS>& l, int b, int from, int to, const float (&A2)[Place<NS>::NC][NS], float (&x)[Place<NS>::NC][NS]) {
#pragma unroll 1
    for (int i = from; i < to; ++i) {
        const int t = BACK ? to - 1 - (i - from) : i;
        bool live = false;
#pragma unroll
        for (int k = 0; k < Place<NS>::NC; ++k) {
            const int c = l.c0 + k;
            if (c >= l.cend) break;
            const float d = (float)delta.row(b, t)[c] + (p.dbias ? p.dbias[c] : 0.f), dt = p.softplus ? softplusf(d) : d;
            float v = (float)in.row(b, t)[c];
            if (!BACK) v *= dt;
            else if (z.p) { const float zv = (float)z.row(b, t)[c]; v *= zv * sigmoidf(zv); }
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int n = l.ng * NS + j;
                if (n >= p.N) break;
                const float a = __builtin_amdgcn_exp2f(dt * A2[k][j]), mv = (float)m.row(b, t)[l.g * p.N + n];
                x[k][j] = BACK ? a * fmaf(mv, v, x[k][j]) : fmaf(a, x[k][j], v * mv);
                live = live || x[k][j] == x[k][j];
            }
        }
        if (!live) break;
    }
}
// x carried over the pieces that walk(carry) goes through: plainly, and where that is not finite (a scan that grows) from reset() again,
// with care, and at last over the frames
template <int NS, typename Walk, typename Reset, typename Frames>
__device__ __forceinline__ void carry_all(float (&x)[Place<NS>::NC][NS], const Walk& walk, const Reset& reset, const Frames& frames) {
    walk(std::false_type{});
    if (all_finite(x)) return;
    reset();
    walk(std::true_type{});
    if (!all_finite(x)) frames();
}

// first launch over a split time axis: a piece alone.  Forward (BACK = false) the state it leaves, from zeros -- the first piece from the
// state it is given; backward the gradient of the state before it, nothing coming from behind.  With it the piece's sum of dt.  Pieces
// that no other one follows (or precedes, backward) are not needed.
template <typename T, int NS, bool BACK, bool GATED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4, 4))) void scan_local_kernel(View<const T> u, View<const T> delta, View<const T> m,
                                                                                                View<const T> z, ScanParams p) {
    // u: dy where BACK;  m: B, or C where BACK
    using L = Place<NS>;
    constexpr int NC = L::NC, TQ = L::TQ, P = L::P, Q = L::Q, SEG = L::SEG, WC = L::WC, ROWS = SEG * 4 * NS;
    __shared__ __align__(16) float bc[2][ROWS];
    const int cb = p.bpg * p.G;
    const int item = (int)(blockIdx.x / cb), b = item / p.chunks, chunk = item - b * p.chunks;
    const L l(p, (int)(blockIdx.x - (unsigned)item * cb));
    const int len = valid_steps(p.lens, b, p.T), nv = (len + SEG - 1) / SEG, last = (nv - 1) / p.spc;
    if (nv == 0 || (BACK ? chunk > last || chunk == 0 : chunk >= last)) return;      // the whole workgroup
    const int s0 = chunk * p.spc, s1 = min(nv, s0 + p.spc);
    float A2[NC][NS], h[NC][NS];
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int c = l.c0 + k, n = l.ng * NS + j;
            const bool on = c < l.cend && n < p.N;
            A2[k][j] = on ? decay2(p.A[(int64_t)c * p.N + n]) : 0.f;
            h[k][j] = !BACK && on && chunk == 0 && p.state_in ? p.state_in[((int64_t)b * p.D + c) * p.N + n] : 0.f;
        }
    const float bias = l.ocv && p.dbias ? p.dbias[l.oc] : 0.f;
    const int first = (BACK ? s1 - 1 : s0) * SEG;
    Walk<const T> wu(u, b, first, l.otp, l.oc, l.ocv), wx(delta, b, first, l.otp, l.oc, l.ocv), wz(z, b, BACK && GATED ? first : 0, l.otp, l.oc, l.ocv);
    const int ms = (int)threadIdx.x / (4 * NS), mn = (int)threadIdx.x % (4 * NS);
    const bool mon = (int)threadIdx.x < ROWS && mn < p.N;
    Walk<const T> wm(m, b, first, ms, l.g * p.N + mn, mon);
    uint32_t un[2][Q], xn[2][Q], zn[2][Q], st[2];
    int ft = first;
    const auto fetch = [&](auto set) {                  // the next segment on the way; outside the utterance nothing
        constexpr int R = decltype(set)::value;
        const auto ru = wu.base(), rx = wx.base(), rz = wz.base();
        st[R] = buf_load<T>(wm.base(), wm.at(0, (unsigned)(ft + ms) < (unsigned)len));
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const bool on = (unsigned)(ft + i * TQ + l.otp) < (unsigned)len;
            un[R][i] = buf_load<T>(ru, wu.at(i * TQ, on));
            xn[R][i] = buf_load<T>(rx, wx.at(i * TQ, on));
            if (BACK && GATED) zn[R][i] = buf_load<T>(rz, wz.at(i * TQ, on));
        }
        constexpr int ON = BACK ? -SEG : SEG;
        ft += ON;
        wu.template move<ON>();
        wx.template move<ON>();
        wm.template move<ON>();
        if (BACK && GATED) wz.template move<ON>();
    };
    float total = 0.f;
    const int n = s1 - s0;
    const auto segment = [&](int k0, auto set) {
        constexpr int R = decltype(set)::value;
        const int seg = BACK ? s1 - 1 - k0 : s0 + k0, t0 = seg * SEG;
        float* buf = bc[R];
        if ((int)threadIdx.x < ROWS) buf[threadIdx.x] = raw_to_float(st[R], T{});
        __syncthreads();
        float in[Q], dt[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const float x = raw_to_float(xn[R][i], T{}) + bias;
            dt[i] = p.softplus ? softplusf(x) : x;
            if (t0 + SEG > len) dt[i] = t0 + i * TQ + l.otp < len ? dt[i] : 0.f;
            in[i] = raw_to_float(un[R][i], T{});
            if (!BACK) in[i] *= dt[i];
            else if (GATED) { const float zc = raw_to_float(zn[R][i], T{}); in[i] *= zc * sigmoidf(zc); }
            total += dt[i];
        }
        fetch(set);
        float mn1[NS];
        load_vec<float, NS>(buf + (BACK ? SEG - 1 : 0) * 4 * NS + l.ng * NS, mn1);
#pragma unroll
        for (int ii = 0; ii < Q; ++ii) {
            const int i = BACK ? Q - 1 - ii : ii;
#pragma unroll
            for (int tt = 0; tt < TQ; ++tt) {
                const int tp = BACK ? TQ - 1 - tt : tt, at = i * TQ + tp, after = BACK ? at - 1 : at + 1;
                float mv[NS];
#pragma unroll
                for (int j = 0; j < NS; ++j) mv[j] = mn1[j];
                if (after >= 0 && after < SEG) load_vec<float, NS>(buf + after * 4 * NS + l.ng * NS, mn1);
                hold_reads();
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const float dtk = bcast(dt[i], tp * NC + k), ink = bcast(in[i], tp * NC + k);
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const float a = __builtin_amdgcn_exp2f(dtk * A2[k][j]);
                        h[k][j] = BACK ? a * fmaf(mv[j], ink, h[k][j]) : fmaf(a, h[k][j], ink * mv[j]);
                    }
                }
            }
        }
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    fetch(even);
    fetch(odd);
    for (int k0 = 0; k0 < n; k0 += 2) {
        segment(k0, even);
        if (k0 + 1 < n) segment(k0 + 1, odd);
    }
    float* out = p.local + local_at<P>(p, b, chunk, l.ctile) + l.lane * 4;
#pragma unroll
    for (int q = 0; q < P / 4; ++q) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = h[(q * 4 + j) / NS][(q * 4 + j) % NS];
        store_vec<float, 4>(out + q * 256, v);
    }
    if constexpr (TQ == 4) total += dpp<kQuadXor1>(total);
    if constexpr (TQ >= 2) total += dpp<kQuadXor2>(total);
    if (l.otp == 0) p.dsum[(((int64_t)b * p.chunks + chunk) * p.ctiles + l.ctile) * WC + l.cl * NC + l.ng] = total;
}

// PIECES: the time axis is split.  The unsplit kernels hold no registers for the carries, and a split one walks one utterance backward
// (520 x 40 x 1000 x 16, unsplit: backward 295 us, as one kernel for both 307; 1 x 8192 x 2048 x 16, split: 296 and 318)
template <typename T, int NS, bool GATED, bool SAVE, bool PIECES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4, 4))) void scan_forward_kernel(View<const T> u, View<const T> delta, View<const T> bm, View<const T> cm, View<const T> z,
                                                           View<T> y, ScanParams p) {
    using L = Place<NS>;
    constexpr int NC = L::NC, TQ = L::TQ, P = L::P, Q = L::Q, SEG = L::SEG, STAGE = L::STAGE;
    __shared__ __align__(16) float bc[2][STAGE];
    const int cb = p.bpg * p.G;
    const int item = (int)(blockIdx.x / cb), b = PIECES ? item / p.chunks : item, chunk = PIECES ? item - b * p.chunks : 0;
    const L l(p, (int)(blockIdx.x - (unsigned)item * cb));
    const int len = valid_steps(p.lens, b, p.T), nv = (len + SEG - 1) / SEG;
    const int s0 = PIECES ? chunk * p.spc : 0, s1 = PIECES ? min(nv, s0 + p.spc) : nv;
    float A2[NC][NS], h[NC][NS];
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int c = l.c0 + k, n = l.ng * NS + j;
            const bool on = c < l.cend && n < p.N;
            A2[k][j] = on ? decay2(p.A[(int64_t)c * p.N + n]) : 0.f;
        }
    const auto first_states = [&](bool given) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int c = l.c0 + k, n = l.ng * NS + j;
                h[k][j] = given && c < l.cend && n < p.N ? p.state_in[((int64_t)b * p.D + c) * p.N + n] : 0.f;
            }
    };
    first_states(chunk == 0 && p.state_in);
    if (PIECES && s0 < nv && chunk > 0)
        carry_all<NS>(h, [&](auto careful) { for (int c = 0; c < chunk; ++c) carry_over<NS, decltype(careful)::value>(p, l, b, c, A2, h); },
                      [&] { first_states(false); },             // (the first piece alone begins with the states that are given)
                      [&] { first_states(p.state_in); over_frames<T, NS, false>(u, delta, bm, View<const T>{}, p, l, b, 0, s0 * SEG, A2, h); });
    const float Dv = l.ocv && p.Dp ? p.Dp[l.oc] : 0.f, bias = l.ocv && p.dbias ? p.dbias[l.oc] : 0.f;
    int ft = s0 * SEG;
    Walk<const T> wu(u, b, ft, l.otp, l.oc, l.ocv), wx(delta, b, ft, l.otp, l.oc, l.ocv), wz(z, b, GATED ? ft : 0, l.otp, l.oc, l.ocv);
    Walk<T> wy(y, b, ft, l.otp, l.oc, l.ocv);
    Walk<const T> wb(bm, b, ft, l.st_s, l.st_at, l.st_s < SEG && !l.st_which), wc(cm, b, ft, l.st_s, l.st_at, l.st_s < SEG && l.st_which);
    // a segment's loads are issued two segments ahead, into one of two sets of registers
    uint32_t un[2][Q], xn[2][Q], zn[2][Q], st[2];
    const auto fetch = [&](auto set) {                  // the next segment; behind the utterance nothing
        constexpr int R = decltype(set)::value;
        const auto ru = wu.base(), rx = wx.base(), rz = wz.base();
        const bool rows = l.st_s < len - ft;
        st[R] = buf_load<T>(wb.base(), wb.at(0, rows)) | buf_load<T>(wc.base(), wc.at(0, rows));
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const bool on = ft + i * TQ + l.otp < len;
            un[R][i] = buf_load<T>(ru, wu.at(i * TQ, on));
            xn[R][i] = buf_load<T>(rx, wx.at(i * TQ, on));
            if (GATED) zn[R][i] = buf_load<T>(rz, wz.at(i * TQ, on));
        }
        ft += SEG;
        wu.template move<SEG>();
        wx.template move<SEG>();
        wb.template move<SEG>();
        wc.template move<SEG>();
        if (GATED) wz.template move<SEG>();
    };
    const auto segment = [&](int seg, auto set) {
        constexpr int R = decltype(set)::value;
        const int t0 = seg * SEG;
        float* buf = bc[R];
        if ((int)threadIdx.x < STAGE) buf[threadIdx.x] = raw_to_float(st[R], T{});
        __syncthreads();            // (the other buffer may still be read by a wave in the segment before)
        float uc[Q], zc[Q], dt[Q], o[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            uc[i] = raw_to_float(un[R][i], T{});
            const float x = raw_to_float(xn[R][i], T{}) + bias;
            if (GATED) zc[i] = raw_to_float(zn[R][i], T{});
            dt[i] = p.softplus ? softplusf(x) : x;
            if (t0 + SEG > len) dt[i] = t0 + i * TQ + l.otp < len ? dt[i] : 0.f;      // the state passes a padding frame
        }
        fetch(set);
        if (SAVE) {
            float* ck = p.ckpt + ckpt_at<P>(p, b, seg, l.ctile) + l.lane * 4;
#pragma unroll
            for (int m = 0; m < P / 4; ++m) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = h[(m * 4 + j) / NS][(m * 4 + j) % NS];
                store_vec<float, 4>(ck + m * 256, v);
            }
        }
        float bn[NS], cn[NS];
        load_vec<float, NS>(buf + l.ng * NS, bn);
        load_vec<float, NS>(buf + 4 * NS + l.ng * NS, cn);
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const float dtu = dt[i] * uc[i];
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int tp = 0; tp < TQ; ++tp) {
                const int after = i * TQ + tp + 1;
                float bv[NS], cv[NS];
#pragma unroll
                for (int j = 0; j < NS; ++j) { bv[j] = bn[j]; cv[j] = cn[j]; }
                if (after < SEG) {
                    load_vec<float, NS>(buf + after * 8 * NS + l.ng * NS, bn);
                    load_vec<float, NS>(buf + after * 8 * NS + 4 * NS + l.ng * NS, cn);
                }
                hold_reads();
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const int q = tp * NC + k;
                    const float dtk = bcast(dt[i], q), dtuk = bcast(dtu, q);
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const float a = __builtin_amdgcn_exp2f(dtk * A2[k][j]);
                        h[k][j] = fmaf(a, h[k][j], dtuk * bv[j]);
                        acc[q] = fmaf(h[k][j], cv[j], acc[q]);
                    }
                }
            }
            o[i] = quad_gather(acc, l.b0, l.b1) + Dv * uc[i];
            if (GATED) o[i] *= zc[i] * sigmoidf(zc[i]);
        }
        const auto ry = wy.base();
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int t = t0 + i * TQ + l.otp;
            buf_store<T>(ry, wy.at(i * TQ, t < p.T), t < len ? o[i] : 0.f);
        }
        wy.template move<SEG>();
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    if (s0 < s1) {
        fetch(even);
        fetch(odd);
        for (int seg = s0; seg < s1; seg += 2) {
            segment(seg, even);
            if (seg + 1 < s1) segment(seg + 1, odd);
        }
    }
    const int end = PIECES ? min(p.T, (s0 + p.spc) * SEG) : p.T;
    for (int t = max(nv, s0) * SEG + l.otp; t < end; t += TQ)
        if (l.ocv) y.row(b, t)[l.oc] = (T)0.f;
    if (!PIECES || chunk == max(nv - 1, 0) / p.spc)
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int c = l.c0 + k, n = l.ng * NS + j;
            if (c < l.cend && n < p.N) p.state_out[((int64_t)b * p.D + c) * p.N + n] = h[k][j];
        }
}

// where reduce_quads leaves a lane's sum in a row of 2 x 4 NS values: behind it (8 NS on, a place nobody reads) where the lane has none
template <int NS> __device__ __forceinline__ int reduced_at(int lane) {
    constexpr int V = 2 * NS;
    int v = (lane >> 5) * (V / 2);
    bool mine = true;
    if (V >= 4) v += ((lane >> 4) & 1) * (V / 4);
    else mine = lane & 16;
    if (V >= 8) v += ((lane >> 3) & 1) * (V / 8);
    else mine = mine && (lane & 8);
    if (V >= 16) v += (lane >> 2) & 1;
    else mine = mine && (lane & 4);
    return (v / NS) * 4 * NS + (lane & 3) * NS + v % NS + (mine ? 0 : 8 * NS);
}
// sum over the 16 quads of a wave of the 2 NS values of each lane (NS of dB, NS of dC): halves are exchanged while there are several
// values, so a step halves the values and adds one bit of the lane to the place
template <int NS> __device__ __forceinline__ float reduce_quads(const float (&v)[2 * NS], const int lane) {
    constexpr int V = 2 * NS;
    float r1[V / 2], r2[(V + 3) / 4];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r1[i] = add_swap32(v[i], v[i + V / 2]);
    if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) r2[i] = add_swap16(r1[i], r1[i + V / 4]);
    } else {
        r2[0] = add_swap16(r1[0], r1[0]);
    }
    const bool b3 = lane & 8, b2 = lane & 4;
    if constexpr (V >= 8) {
        float r3[V / 8];
#pragma unroll
        for (int i = 0; i < V / 8; ++i) r3[i] = (b3 ? r2[i + V / 8] : r2[i]) + dpp<kRowRor8>(b3 ? r2[i] : r2[i + V / 8]);
        if constexpr (V >= 16)      // the swizzle: lane ^ 4
            return (b2 ? r3[1] : r3[0]) + __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, b2 ? r3[0] : r3[1]), 0x101F));
        else
            return r3[0] + dpp<kRowShr4>(r3[0]);          // complete in the lanes with bit 2 set
    } else {
        const float r = r2[0] + dpp<kRowRor8>(r2[0]);
        return r + dpp<kRowShr4>(r);
    }
}

template <typename T, int NS, bool GATED, bool PIECES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void scan_backward_kernel(View<const T> u, View<const T> delta, View<const T> bm, View<const T> cm, View<const T> z,
                                                               View<const T> dy, View<T> du, View<T> ddelta, View<T> dz, ScanParams p) {
    using L = Place<NS>;
    constexpr int NC = L::NC, TQ = L::TQ, P = L::P, Q = L::Q, WC = L::WC, SEG = L::SEG, STAGE = L::STAGE;
    constexpr bool KEEP = NS != 2;                      // the segment's states too, not a and e alone: a multiply-add less, where registers are left
    __shared__ __align__(16) float bc[2][STAGE];
    __shared__ float red[2][4][SEG][16 * NS];           // per frame 8 NS sums and 8 NS places nobody reads
    const int cb = p.bpg * p.G;
    const int item = (int)(blockIdx.x / cb), cblk = (int)(blockIdx.x - (unsigned)item * cb), bg = PIECES ? item / p.chunks : item, chunk = PIECES ? item - bg * p.chunks : 0;
    const L l(p, cblk);
    const int red_at = reduced_at<NS>(l.lane);
    float A2[NC][NS], dA[NC][NS];
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int c = l.c0 + k, n = l.ng * NS + j;
            A2[k][j] = c < l.cend && n < p.N ? decay2(p.A[(int64_t)c * p.N + n]) : 0.f;
            dA[k][j] = 0.f;
        }
    const float Dv = l.ocv && p.Dp ? p.Dp[l.oc] : 0.f, bias = l.ocv && p.dbias ? p.dbias[l.oc] : 0.f;
    float dD = 0.f, dbias = 0.f;
    int turn = 0;
    float* flush_at = nullptr;                  // where the sums waiting in red[turn ^ 1] go
    auto flush = [&](const float (*rd)[SEG][16 * NS]) {
        const int i = threadIdx.x, s = i / (8 * NS), at = i % (8 * NS);
        if (i < STAGE) flush_at[i] = ((rd[0][s][at] + rd[1][s][at]) + rd[2][s][at]) + rd[3][s][at];
    };
    const int b_end = PIECES ? bg + 1 : min(p.B, (bg + 1) * p.per_bg);       // (an utterance a group where it is in pieces)
    for (int b = PIECES ? bg : bg * p.per_bg; b < b_end; ++b) {
        const int len = valid_steps(p.lens, b, p.T), nv = (len + SEG - 1) / SEG;
        float carry[NC][NS];
        const auto last_gradients = [&] {
#pragma unroll
            for (int k = 0; k < NC; ++k)
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    const int c = l.c0 + k, n = l.ng * NS + j;
                    carry[k][j] = p.dlast && c < l.cend && n < p.N ? p.dlast[((int64_t)b * p.D + c) * p.N + n] : 0.f;
                }
        };
        last_gradients();
        const int s0 = PIECES ? chunk * p.spc : 0, s1 = PIECES ? min(nv, s0 + p.spc) : nv, end = PIECES ? min(p.T, (s0 + p.spc) * SEG) : p.T;
        if (PIECES && s1 < nv)
            carry_all<NS>(carry, [&](auto careful) { for (int c = (nv - 1) / p.spc; c > chunk; --c) carry_over<NS, decltype(careful)::value>(p, l, b, c, A2, carry); },
                          last_gradients, [&] { last_gradients(); over_frames<T, NS, true>(dy, delta, cm, GATED ? z : View<const T>{}, p, l, b, s1 * SEG, len, A2, carry); });
        for (int t = max(nv, s0) * SEG + l.otp; t < end; t += TQ)
            if (l.ocv) {
                du.row(b, t)[l.oc] = (T)0.f;
                ddelta.row(b, t)[l.oc] = (T)0.f;
                if (GATED) dz.row(b, t)[l.oc] = (T)0.f;
            }
        const Walk<const T> wu(u, b, 0, l.otp, l.oc, l.ocv), wx(delta, b, 0, l.otp, l.oc, l.ocv), wz(z, b, 0, l.otp, l.oc, l.ocv), wg(dy, b, 0, l.otp, l.oc, l.ocv);
        const Walk<T> wdu(du, b, 0, l.otp, l.oc, l.ocv), wdx(ddelta, b, 0, l.otp, l.oc, l.ocv), wdz(dz, b, 0, l.otp, l.oc, l.ocv);
        const Walk<const T> wb(bm, b, 0, l.st_s, l.st_at, l.st_s < SEG && !l.st_which), wc(cm, b, 0, l.st_s, l.st_at, l.st_s < SEG && l.st_which);
        uint32_t un[Q], xn[Q], zn[Q], gn[Q], st;
        float hn[P];
        const auto fetch = [&](int of) {                // before the first segment: the first one again
            const int seg = max(of, s0), t0 = seg * SEG;
            const auto ru = wu.base(t0), rx = wx.base(t0), rz = wz.base(t0), rg = wg.base(t0);
            const bool rows = l.st_s < len - t0;
            st = buf_load<T>(wb.base(t0), wb.at(0, rows)) | buf_load<T>(wc.base(t0), wc.at(0, rows));
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const bool on = t0 + i * TQ + l.otp < len;
                un[i] = buf_load<T>(ru, wu.at(i * TQ, on));
                xn[i] = buf_load<T>(rx, wx.at(i * TQ, on));
                gn[i] = buf_load<T>(rg, wg.at(i * TQ, on));
                if (GATED) zn[i] = buf_load<T>(rz, wz.at(i * TQ, on));
            }
            const float* ck = p.ckpt + ckpt_at<P>(p, b, seg, l.ctile) + l.lane * 4;
#pragma unroll
            for (int m = 0; m < P / 4; ++m) load_vec<float, 4>(ck + m * 256, hn + m * 4);
        };
        if (s0 < s1) fetch(s1 - 1);
        for (int seg = s1 - 1; seg >= s0; --seg) {
            float* buf = bc[turn];
            if ((int)threadIdx.x < STAGE) buf[threadIdx.x] = raw_to_float(st, T{});
            __syncthreads();                    // B and C are in; the sums of the segment before are complete
            if (flush_at) flush(red[turn ^ 1]);
            flush_at = p.part_bc + ((((int64_t)(cblk - l.g * p.bpg) * p.B + b) * p.nseg + seg) * p.G + l.g) * STAGE;
            const int t0 = seg * SEG;
            const bool full = t0 + SEG <= len;
            float uc[Q], xc[Q], zc[Q], gc[Q], dt[Q], h[NC][NS], odu[Q], odx[Q], odz[Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                uc[i] = raw_to_float(un[i], T{});
                xc[i] = raw_to_float(xn[i], T{}) + bias;
                gc[i] = raw_to_float(gn[i], T{});
                if (GATED) zc[i] = raw_to_float(zn[i], T{});
                dt[i] = p.softplus ? softplusf(xc[i]) : xc[i];
                if (!full) dt[i] = t0 + i * TQ + l.otp < len ? dt[i] : 0.f;
            }
#pragma unroll
            for (int m = 0; m < P; ++m) h[m / NS][m % NS] = hn[m];
            fetch(seg - 1);
            float a[SEG][NC][NS], e[SEG][NC][NS], hs[KEEP ? SEG : 1][NC][NS], bn[NS], cn[NS];
            load_vec<float, NS>(buf + l.ng * NS, bn);
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const float dtu = dt[i] * uc[i];
#pragma unroll
                for (int tp = 0; tp < TQ; ++tp) {
                    const int s = i * TQ + tp;
                    float bv[NS];
#pragma unroll
                    for (int j = 0; j < NS; ++j) bv[j] = bn[j];
                    load_vec<float, NS>(buf + min(s + 1, SEG - 1) * 8 * NS + l.ng * NS, bn);
                    if (s + 1 == SEG) load_vec<float, NS>(buf + s * 8 * NS + 4 * NS + l.ng * NS, cn);
                    hold_reads();
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        const float dtk = bcast(dt[i], tp * NC + k), dtuk = bcast(dtu, tp * NC + k);
#pragma unroll
                        for (int j = 0; j < NS; ++j) {
                            a[s][k][j] = __builtin_amdgcn_exp2f(dtk * A2[k][j]);
                            e[s][k][j] = a[s][k][j] * h[k][j];
                            h[k][j] = fmaf(dtuk, bv[j], e[s][k][j]);
                            if (KEEP) hs[s][k][j] = h[k][j];
                        }
                    }
                }
            }
#pragma unroll
            for (int i = Q - 1; i >= 0; --i) {
                const float dtu = dt[i] * uc[i];
                float sg = 0.f, dyp = gc[i];
                if (GATED) { sg = sigmoidf(zc[i]); dyp *= zc[i] * sg; }
                float s1[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f}, sy[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int tp = TQ - 1; tp >= 0; --tp) {
                    const int s = i * TQ + tp;
                    float bv[NS], cv[NS], sums[2 * NS];
#pragma unroll
                    for (int j = 0; j < NS; ++j) { bv[j] = bn[j]; cv[j] = cn[j]; }
                    if (s > 0) {
                        load_vec<float, NS>(buf + (s - 1) * 8 * NS + l.ng * NS, bn);
                        load_vec<float, NS>(buf + (s - 1) * 8 * NS + 4 * NS + l.ng * NS, cn);
                    }
                    hold_reads();
#pragma unroll
                    for (int j = 0; j < 2 * NS; ++j) sums[j] = 0.f;
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        const int q = tp * NC + k;
                        const float dtk = bcast(dt[i], q), dtuk = bcast(dtu, q), dyk = bcast(dyp, q);
#pragma unroll
                        for (int j = 0; j < NS; ++j) {
                            const float dh = fmaf(cv[j], dyk, carry[k][j]), hv = KEEP ? hs[s][k][j] : fmaf(dtuk, bv[j], e[s][k][j]), de = dh * e[s][k][j];
                            sums[j] = fmaf(dtuk, dh, sums[j]);
                            sums[NS + j] = fmaf(dyk, hv, sums[NS + j]);
                            s1[q] = fmaf(dh, bv[j], s1[q]);
                            s2[q] = fmaf(A2[k][j], de, s2[q]);
                            if (GATED) sy[q] = fmaf(cv[j], hv, sy[q]);
                            dA[k][j] = fmaf(dtk, de, dA[k][j]);
                            carry[k][j] = a[s][k][j] * dh;
                        }
                    }
                    red[turn][l.wv][s][red_at] = reduce_quads<NS>(sums, l.lane);
                }
                const float ddtu = quad_gather(s1, l.b0, l.b1), ddec = quad_gather(s2, l.b0, l.b1) * kLn2;
                float dx = ddec + uc[i] * ddtu;
                if (p.softplus) dx *= sigmoidf(xc[i]);
                if (!full) dx = t0 + i * TQ + l.otp < len ? dx : 0.f;
                odu[i] = dt[i] * ddtu + Dv * dyp;
                odx[i] = dx;
                dbias += dx;
                dD += dyp * uc[i];
                if (GATED) odz[i] = gc[i] * (quad_gather(sy, l.b0, l.b1) + Dv * uc[i]) * sg * (1.f + zc[i] * (1.f - sg));
            }
            const auto rdu = wdu.base(t0), rdx = wdx.base(t0), rdz = wdz.base(t0);
            if (!full)               // zeros for padding, also where an infinite state or gradient passes it
#pragma unroll
                for (int i = 0; i < Q; ++i)
                    if (t0 + i * TQ + l.otp >= len) odu[i] = odz[i] = 0.f;
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const bool on = t0 + i * TQ + l.otp < p.T;
                buf_store<T>(rdu, wdu.at(i * TQ, on), odu[i]);
                buf_store<T>(rdx, wdx.at(i * TQ, on), odx[i]);
                if (GATED) buf_store<T>(rdz, wdz.at(i * TQ, on), odz[i]);
            }
            turn ^= 1;
        }
        if (p.dstate && (!PIECES || chunk == 0))
#pragma unroll
            for (int k = 0; k < NC; ++k)
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    const int c = l.c0 + k, n = l.ng * NS + j;
                    if (c < l.cend && n < p.N) p.dstate[((int64_t)b * p.D + c) * p.N + n] = carry[k][j];
                }
    }
    __syncthreads();
    if (flush_at) flush(red[turn ^ 1]);
    float* out = p.part_a + ((int64_t)item * p.ctiles + l.ctile) * (64 * P + 2 * WC);
#pragma unroll
    for (int m = 0; m < P / 4; ++m) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = dA[(m * 4 + j) / NS][(m * 4 + j) % NS];
        store_vec<float, 4>(out + (m * 64 + l.lane) * 4, v);
    }
    if constexpr (TQ == 4) { dD += dpp<kQuadXor1>(dD); dbias += dpp<kQuadXor1>(dbias); }
    if constexpr (TQ >= 2) { dD += dpp<kQuadXor2>(dD); dbias += dpp<kQuadXor2>(dbias); }
    if (l.otp == 0) {
        out[64 * P + l.cl * NC + l.ng] = dD;
        out[64 * P + WC + l.cl * NC + l.ng] = dbias;
    }
}

// sum of n values `stride` apart, in order, eight loads in flight
__device__ __forceinline__ float strided_sum(const float* __restrict__ src, int64_t stride, int n) {
    float a = 0.f;
    int k = 0;
    for (; k + 8 <= n; k += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = src[(k + i) * stride];
#pragma unroll
        for (int i = 0; i < 8; ++i) a += v[i];
    }
    for (; k < n; ++k) a += src[k * stride];
    return a;
}

// the second launch of the backward pass: workgroups [0, nb_bc) add dB and dC over the workgroups of a group, the others dA, dD and
// the bias' gradient over the groups of utterances
template <typename T, int NS>
__global__ __launch_bounds__(256) void scan_reduce_kernel(T* __restrict__ dB, T* __restrict__ dC, float* __restrict__ dA, float* __restrict__ dD,
                                                          float* __restrict__ dbias, ScanParams p, int nb_bc) {
    using L = Place<NS>;
    constexpr int P = L::P, WC = L::WC, NC = L::NC, SEG = L::SEG, STAGE = L::STAGE;
    if ((int)blockIdx.x < nb_bc) {
        // fewer than 2^32 of them (the launch's limit), B's first
        const unsigned gn = (unsigned)p.G * (unsigned)p.N, half = (unsigned)p.B * (unsigned)p.T * gn;
        const unsigned i = blockIdx.x * 256 + threadIdx.x;
        if (i >= 2 * half) return;
        const int which = i >= half;
        const unsigned o = i - (which ? half : 0), bt = o / gn, r = o - bt * gn;
        const int g = (int)(r / (unsigned)p.N), n = (int)(r - (unsigned)g * (unsigned)p.N), b = (int)(bt / (unsigned)p.T), t = (int)(bt - (unsigned)b * (unsigned)p.T);
        float a = 0.f;
        if (t < valid_steps(p.lens, b, p.T)) {
            const float* src = p.part_bc + (((int64_t)b * p.nseg + t / SEG) * p.G + g) * STAGE + (t % SEG) * 8 * NS + which * 4 * NS + n;
            a = strided_sum(src, (int64_t)p.B * p.nseg * p.G * STAGE, p.bpg);
        }
        (which ? dC : dB)[o] = (T)a;
        return;
    }
    // 32 results x 8 lanes: lane k adds parts k, k + 8, ... and the eight sums are added in order
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t i = (int64_t)(blockIdx.x - nb_bc) * 32 + lane, da = (int64_t)p.D * p.N;
    const bool on = i < da + 2 * (int64_t)p.D;
    const int c = on ? (int)(i < da ? i / p.N : (i - da) % p.D) : 0, n = (int)(i % p.N);
    const int g = c / p.Dg, cg = c - g * p.Dg, tg = cg / WC, cw = cg % WC, parts = p.nbg * p.chunks;
    const int64_t row = (int64_t)(g * p.bpg * 4 + tg) * (64 * P + 2 * WC), stride = (int64_t)p.ctiles * (64 * P + 2 * WC);
    int64_t at;
    if (i < da) {
        const int lane_of = cw / NC * 4 + n / NS, m = cw % NC * NS + n % NS;
        at = (m / 4 * 64 + lane_of) * 4 + m % 4;
    } else
        at = 64 * P + (i - da >= p.D ? WC : 0) + cw;
    red[k][lane] = on ? strided_sum(p.part_a + row + at + k * stride, 8 * stride, (parts - k + 7) / 8) : 0.f;
    __syncthreads();
    if (k || !on) return;
    float v = red[0][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) v += red[w][lane];
    if (i < da) dA[i] = v;
    else if (i - da < p.D) dD[c] = v;
    else dbias[c] = v;
}

// one frame of every utterance, the state moved on in place: a quad per channel, NS neighbouring states per lane; VEC: N in whole
// vectors of min(NS, 4) states and everything aligned for them (321 x 2102 x 24: 27 us, state by state 75).  Bound by the state's
// bytes, in and out
template <typename T, int NS, bool VEC>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* __restrict__ u, int64_t ldu, const T* __restrict__ delta, int64_t ldd, const T* __restrict__ bm,
                                                        int64_t ldb, const T* __restrict__ cm, int64_t ldc, const T* __restrict__ z, int64_t ldz,
                                                        T* __restrict__ y, int64_t ldy, ScanParams p) {
    const unsigned item = blockIdx.x * 64 + threadIdx.x / 4;      // B D < 2^31
    const int ng = threadIdx.x & 3;
    if (item >= (unsigned)p.B * (unsigned)p.D) return;             // whole quads leave
    const int b = (int)(item / (unsigned)p.D), c = (int)(item - (unsigned)b * (unsigned)p.D), g = p.G == 1 ? 0 : c / p.Dg;
    const float uv = (float)u[b * ldu + c];
    float dt = (float)delta[b * ldd + c] + (p.dbias ? p.dbias[c] : 0.f);
    if (p.softplus) dt = softplusf(dt);
    const float dtu = dt * uv;
    float* h = p.state_out + (int64_t)item * p.N;
    const T* br = bm + b * ldb + (int64_t)g * p.N;
    const T* cr = cm + b * ldc + (int64_t)g * p.N;
    float acc = 0.f, hv[NS], av[NS], bv[NS], cv[NS];
    constexpr int W = NS < 4 ? NS : 4;
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < NS; j += W) {
            const int n = ng * NS + j;
            if (n < p.N) {
                load_vec<float, W>(h + n, hv + j);
                load_vec<float, W>(p.A + (int64_t)c * p.N + n, av + j);
                load_vec<T, W>(br + n, bv + j);
                load_vec<T, W>(cr + n, cv + j);
            } else
#pragma unroll
                for (int i = 0; i < W; ++i) hv[j + i] = av[j + i] = bv[j + i] = cv[j + i] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int n = ng * NS + j;
            const bool on = n < p.N;
            hv[j] = on ? h[n] : 0.f;
            av[j] = on ? p.A[(int64_t)c * p.N + n] : 0.f;
            bv[j] = on ? (float)br[n] : 0.f;
            cv[j] = on ? (float)cr[n] : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        hv[j] = fmaf(__builtin_amdgcn_exp2f(dt * decay2(av[j])), hv[j], dtu * bv[j]);
        acc = fmaf(hv[j], cv[j], acc);
    }
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < NS; j += W)
            if (ng * NS + j < p.N) store_vec<float, W>(h + ng * NS + j, hv + j);
    } else
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (ng * NS + j < p.N) h[ng * NS + j] = hv[j];
    acc += dpp<kQuadXor1>(acc);
    acc += dpp<kQuadXor2>(acc);
    if (ng == 0) {
        float o = acc + (p.Dp ? p.Dp[c] : 0.f) * uv;
        if (z) {
            const float zv = (float)z[b * ldz + c];
            o *= zv * sigmoidf(zv);
        }
        y[b * ldy + c] = (T)o;
    }
}

int states_per_lane(int n) { return n <= 4 ? 1 : (n <= 8 ? 2 : (n <= 16 ? 4 : 8)); }

constexpr int kMinPiece = 8;           // segments of a piece, at least

struct Plan { int ns, nc, nseg, tpg, bpg, ctiles, nbg, per_bg, chunks, spc; int64_t ckpt, part_bc, part_a, local, dsum; };

Plan plan_of(int64_t B, int64_t T, int D, int N, int G, bool bwd) {
    Plan q{};
    q.ns = states_per_lane(N);
    q.nc = channels_per_quad(q.ns);
    const int Dg = D / G, P = q.ns * q.nc, WC = 16 * q.nc;
    const int seg = segment_frames(q.ns);
    q.nseg = cdiv(T, seg);
    q.tpg = cdiv(Dg, WC);
    q.bpg = cdiv(q.tpg, 4);
    q.ctiles = q.bpg * G * 4;
    q.ckpt = B * q.nseg * q.ctiles * 64 * P;
    // backward: groups of utterances for about 1024 workgroups, two rounds of the 512 that are resident (two waves per SIMD); rounding
    // the group's size down can leave a few for a third round
    const int64_t want = std::max<int64_t>(1, cdiv(1024, q.bpg * G));
    q.per_bg = (int)std::max<int64_t>(1, B / want);
    q.nbg = cdiv(B, q.per_bg);
    // (workgroups are whole, four waves: 64 channels of 16 states, 256 of up to 4.  A group of fewer channels runs waves that own none,
    // and their states are kept too: 520 x 2000 x 16 channels of 4 states take 1.07 GB of checkpoints)
    // a time axis in pieces, where the utterances and channels alone are too few waves: the first launch costs 7 / 8 of the work once
    // more forward and a third of it backward.  512 frames x 2048 channels x 16 states, 768 waves: forward 60 against 70 us, 1024
    // waves: forward 76 against 72, backward 172 against 180 us
    const int64_t waves = B * q.tpg * G;
    q.chunks = 1;
    if (B > 0 && waves <= (bwd ? 1024 : 768) && q.nseg >= 2 * kMinPiece)
        q.chunks = (int)std::min<int64_t>(q.nseg / kMinPiece, (4096 + waves - 1) / waves);
    q.spc = std::max(1, cdiv(q.nseg, q.chunks));
    q.chunks = std::max(1, cdiv(q.nseg, q.spc));
    if (q.chunks > 1) {      // the pieces' launches go by utterance (so few waves make groups of one anyway)
        q.per_bg = 1;
        q.nbg = (int)B;
    }
    q.local = q.chunks > 1 ? B * q.chunks * q.ctiles * 64 * P : 0;
    q.dsum = q.chunks > 1 ? B * q.chunks * q.ctiles * WC : 0;
    q.part_bc = (int64_t)q.bpg * B * q.nseg * G * seg * 8 * q.ns;
    q.part_a = (int64_t)q.nbg * q.chunks * q.ctiles * (64 * P + 2 * WC);
    return q;
}

bool sizes_ok(int64_t B, int64_t T, int64_t D, int64_t N, int64_t G) {
    return B >= 0 && T >= 0 && B * T < ((int64_t)1 << 31) - 65536 && D >= 1 && D <= 1 << 20 && N >= 1 && N <= kMaxStates && G >= 1 && D % G == 0 &&
           B * D < (int64_t)1 << 31;
}

int check(const adn_scan_args* a, const char* who, bool backward) {
    ADN_CHECK(a, ADN_ERR_INVALID, std::string(who) + ": null arguments");
    ADN_CHECK(a->dtype == ADN_DTYPE_F32 || a->dtype == ADN_DTYPE_BF16, ADN_ERR_INVALID, std::string(who) + ": dtype is ADN_DTYPE_F32 or ADN_DTYPE_BF16");
    ADN_CHECK(a->batch >= 0 && a->steps >= 0 && (int64_t)a->batch * a->steps < ((int64_t)1 << 31) - 65536, ADN_ERR_INVALID, std::string(who) + ": bad (batch, steps)");
    ADN_CHECK(a->states >= 1 && a->states <= kMaxStates, ADN_ERR_INVALID, std::string(who) + ": states outside 1 .. 32");
    ADN_CHECK(a->channels >= 1 && a->channels <= 1 << 20 && a->groups >= 1 && a->channels % a->groups == 0, ADN_ERR_INVALID,
              std::string(who) + ": channels outside 1 .. 2^20 or not a multiple of groups");
    ADN_CHECK(sizes_ok(a->batch, a->steps, a->channels, a->states, a->groups), ADN_ERR_INVALID, std::string(who) + ": batch * channels too large");
    ADN_CHECK(a->A, ADN_ERR_INVALID, std::string(who) + ": null A");
    const int e = a->dtype == ADN_DTYPE_BF16 ? 2 : 4;
    // 31-bit offsets within a segment: seven frames on, and a channel
    const auto far = [&](const adn_seq& t) { return a->steps > 1 && t.data && (t.stride_t < 0 || t.stride_t >= (int64_t)1 << 26); };
    ADN_CHECK(!far(a->u) && !far(a->delta) && !far(a->b) && !far(a->c) && !far(a->z) && !far(a->y) && !far(a->dy) && !far(a->du) && !far(a->ddelta) && !far(a->dz),
              ADN_ERR_INVALID, std::string(who) + ": a frame stride outside 0 .. 2^26");
    if ((int64_t)a->batch * a->steps > 0) {
        ADN_CHECK(seq_ok(a->u, e) && seq_ok(a->delta, e) && seq_ok(a->b, e) && seq_ok(a->c, e), ADN_ERR_INVALID, std::string(who) + ": null or misaligned tensor");
        ADN_CHECK(!a->z.data || seq_ok(a->z, e), ADN_ERR_INVALID, std::string(who) + ": misaligned gate");
        if (!backward) ADN_CHECK(seq_ok(a->y, e), ADN_ERR_INVALID, std::string(who) + ": null or misaligned y");
        else ADN_CHECK(seq_ok(a->dy, e) && seq_ok(a->du, e) && seq_ok(a->ddelta, e) && (!a->z.data || seq_ok(a->dz, e)), ADN_ERR_INVALID,
                       std::string(who) + ": null or misaligned gradient");
    }
    return ADN_OK;
}

ScanParams params(const adn_scan_args& a, const Plan& q) {
    ScanParams p{};
    p.lens = a.lens; p.A = a.A; p.Dp = a.D; p.dbias = a.delta_bias; p.state_in = a.state; p.state_out = a.state_out; p.ckpt = a.checkpoints;
    p.dlast = a.dlast; p.dstate = a.dstate;
    p.B = a.batch; p.T = a.steps; p.D = a.channels; p.N = a.states; p.G = a.groups; p.Dg = a.channels / a.groups;
    p.nseg = q.nseg; p.bpg = q.bpg; p.ctiles = q.ctiles; p.nbg = q.nbg; p.per_bg = q.per_bg;
    p.chunks = q.chunks; p.spc = q.spc;
    p.softplus = a.softplus;
    return p;
}

// go(...) with every truth value as a type
template <typename F, typename... Rest> void choose(const F& go, bool first, Rest... rest) {
    if constexpr (sizeof...(rest) == 0) {
        if (first) go(std::true_type{});
        else go(std::false_type{});
    } else {
        if (first) choose([&](auto... t) { go(std::true_type{}, t...); }, rest...);
        else choose([&](auto... t) { go(std::false_type{}, t...); }, rest...);
    }
}

template <typename T, int NS> int forward(const adn_scan_args& a, const ScanParams& p, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.B * p.chunks * p.bpg * p.G));
    if (p.chunks > 1)
        hipLaunchKernelGGL((scan_local_kernel<T, NS, false, false>), grid, dim3(256), 0, s, cview<T>(a.u), cview<T>(a.delta), cview<T>(a.b), View<const T>{}, p);
    const auto go = [&](auto gated, auto save, auto pieces) {
        hipLaunchKernelGGL((scan_forward_kernel<T, NS, decltype(gated)::value, decltype(save)::value, decltype(pieces)::value>), grid, dim3(256), 0, s, cview<T>(a.u),
                           cview<T>(a.delta), cview<T>(a.b), cview<T>(a.c), cview<T>(a.z), view<T>(a.y), p);
    };
    choose(go, a.z.data != nullptr, p.ckpt != nullptr, p.chunks > 1);
    ADN_HIP_CHECK(hipGetLastError());
    return ADN_OK;
}

template <typename T, int NS> int backward(const adn_scan_args& a, const ScanParams& p, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.nbg * p.chunks * p.bpg * p.G));
    if (p.chunks > 1) {      // (one utterance per group then: the pieces' grid is B x chunks)
        if (a.z.data) hipLaunchKernelGGL((scan_local_kernel<T, NS, true, true>), grid, dim3(256), 0, s, cview<T>(a.dy), cview<T>(a.delta), cview<T>(a.c), cview<T>(a.z), p);
        else hipLaunchKernelGGL((scan_local_kernel<T, NS, true, false>), grid, dim3(256), 0, s, cview<T>(a.dy), cview<T>(a.delta), cview<T>(a.c), View<const T>{}, p);
    }
    const auto go = [&](auto gated, auto pieces) {
        hipLaunchKernelGGL((scan_backward_kernel<T, NS, decltype(gated)::value, decltype(pieces)::value>), grid, dim3(256), 0, s, cview<T>(a.u), cview<T>(a.delta),
                           cview<T>(a.b), cview<T>(a.c), cview<T>(a.z), cview<T>(a.dy), view<T>(a.du), view<T>(a.ddelta), view<T>(a.dz), p);
    };
    if (p.B > 0) {
        choose(go, a.z.data != nullptr, p.chunks > 1);
        ADN_HIP_CHECK(hipGetLastError());
    }
    const int64_t bc = (int64_t)p.B * p.T * p.G * p.N * 2, rest = (int64_t)p.D * (p.N + 2);
    const int64_t nb_bc = (bc + 255) / 256;
    hipLaunchKernelGGL((scan_reduce_kernel<T, NS>), dim3((unsigned)(nb_bc + (rest + 31) / 32)), dim3(256), 0, s, static_cast<T*>(a.dB), static_cast<T*>(a.dC),
                       a.dA, a.dD, a.ddelta_bias, p, (int)nb_bc);
    ADN_HIP_CHECK(hipGetLastError());
    return ADN_OK;
}

template <typename T, int NS> int step(const adn_scan_args& a, const ScanParams& p, hipStream_t s) {
    const int64_t items = (int64_t)p.B * p.D;
    const int e = sizeof(T);
    constexpr int W = NS < 4 ? NS : 4;
    const auto rows = [&](const adn_seq& t) { return ptr_aligned(t.data, W * e) && t.stride_b % W == 0; };
    const bool vec = p.N % W == 0 && ptr_aligned(p.A, 16) && ptr_aligned(p.state_out, 16) && rows(a.b) && rows(a.c);
#define ADN_SCAN_GO(VEC)                                                                                                                           \
    hipLaunchKernelGGL((scan_step_kernel<T, NS, VEC>), dim3((unsigned)((items + 63) / 64)), dim3(256), 0, s, static_cast<const T*>(a.u.data), a.u.stride_b, \
                       static_cast<const T*>(a.delta.data), a.delta.stride_b, static_cast<const T*>(a.b.data), a.b.stride_b, static_cast<const T*>(a.c.data), \
                       a.c.stride_b, static_cast<const T*>(a.z.data), a.z.stride_b, static_cast<T*>(a.y.data), a.y.stride_b, p)
    if (vec) ADN_SCAN_GO(true);
    else ADN_SCAN_GO(false);
#undef ADN_SCAN_GO
    ADN_HIP_CHECK(hipGetLastError());
    return ADN_OK;
}

enum Pass { kForward, kBackward, kStep };
template <typename T, Pass PASS, int NS> int go(const adn_scan_args& a, const ScanParams& p, hipStream_t s) {
    if constexpr (PASS == kForward) return forward<T, NS>(a, p, s);
    else if constexpr (PASS == kBackward) return backward<T, NS>(a, p, s);
    else return step<T, NS>(a, p, s);
}
template <typename T, Pass PASS> int by_states(const adn_scan_args& a, const ScanParams& p, int ns, hipStream_t s) {
    switch (ns) {
        case 1: return go<T, PASS, 1>(a, p, s);
        case 2: return go<T, PASS, 2>(a, p, s);
        case 4: return go<T, PASS, 4>(a, p, s);
        default: return go<T, PASS, 8>(a, p, s);
    }
}
template <Pass PASS> int dispatch(const adn_scan_args& a, const ScanParams& p, int ns, hipStream_t s) {
    return a.dtype == ADN_DTYPE_BF16 ? by_states<__bf16, PASS>(a, p, ns, s) : by_states<float, PASS>(a, p, ns, s);
}

}  // namespace
}  // namespace seq
}  // namespace adn

using namespace adn;
using namespace adn::seq;

extern "C" int64_t adn_op_selective_scan_checkpoints(int32_t batch, int32_t steps, int32_t channels, int32_t states, int32_t groups) {
    if (!sizes_ok(batch, steps, channels, states, groups)) return -1;
    return plan_of(batch, steps, channels, states, groups, false).ckpt;
}

extern "C" int64_t adn_op_selective_scan_workspace(int32_t batch, int32_t steps, int32_t channels, int32_t states, int32_t groups, int32_t backward) {
    if (!sizes_ok(batch, steps, channels, states, groups)) return -1;
    const Plan q = plan_of(batch, steps, channels, states, groups, backward != 0);
    return q.local + q.dsum + (backward ? q.part_a + q.part_bc : 0);
}

extern "C" int adn_op_selective_scan_forward(const adn_scan_args* a, void* hip_stream) {
    ADN_TRY(check(a, "adn_op_selective_scan_forward", false));
    if (a->batch == 0) return ADN_OK;
    ADN_CHECK(a->state_out && a->state_out != a->state, ADN_ERR_INVALID, "adn_op_selective_scan_forward: state_out is null or the state that is read");
    const Plan q = plan_of(a->batch, a->steps, a->channels, a->states, a->groups, false);
    ADN_CHECK(!a->checkpoints || (ptr_aligned(a->checkpoints, 16) && a->checkpoint_floats >= q.ckpt), ADN_ERR_INVALID,
              "adn_op_selective_scan_forward: checkpoints smaller than adn_op_selective_scan_checkpoints() floats, or not on 16 bytes");
    ADN_CHECK(q.local == 0 || (a->workspace && ptr_aligned(a->workspace, 16) && a->workspace_floats >= q.local + q.dsum), ADN_ERR_INVALID,
              "adn_op_selective_scan_forward: workspace smaller than adn_op_selective_scan_workspace() floats, or not on 16 bytes");
    ADN_CHECK(grid_ok((int64_t)a->batch * q.chunks * q.bpg * a->groups), ADN_ERR_INVALID, "adn_op_selective_scan_forward: batch too large");
    ScanParams p = params(*a, q);
    p.local = a->workspace;
    p.dsum = a->workspace + q.local;
    return dispatch<kForward>(*a, p, q.ns, static_cast<hipStream_t>(hip_stream));
}

extern "C" int adn_op_selective_scan_backward(const adn_scan_args* a, void* hip_stream) {
    ADN_TRY(check(a, "adn_op_selective_scan_backward", true));
    ADN_CHECK(a->dA && a->dD && a->ddelta_bias, ADN_ERR_INVALID, "adn_op_selective_scan_backward: null gradient");
    const int64_t frames = (int64_t)a->batch * a->steps;
    ADN_CHECK(frames == 0 || (a->dB && a->dC), ADN_ERR_INVALID, "adn_op_selective_scan_backward: null gradient");
    const Plan q = plan_of(a->batch, a->steps, a->channels, a->states, a->groups, true);
    ADN_CHECK(q.ckpt == 0 || (a->checkpoints && ptr_aligned(a->checkpoints, 16) && a->checkpoint_floats >= q.ckpt), ADN_ERR_INVALID,
              "adn_op_selective_scan_backward: needs the checkpoints of the forward pass");
    const int64_t need = q.part_a + q.part_bc + q.local + q.dsum;
    ADN_CHECK(need == 0 || (a->workspace && ptr_aligned(a->workspace, 16) && a->workspace_floats >= need), ADN_ERR_INVALID,
              "adn_op_selective_scan_backward: workspace smaller than adn_op_selective_scan_workspace() floats, or not on 16 bytes");
    const int64_t sums = (int64_t)a->batch * a->steps * a->groups * a->states * 2 + (int64_t)a->channels * (a->states + 2) * 8;
    ADN_CHECK(grid_ok((int64_t)q.nbg * q.chunks * q.bpg * a->groups) && grid_ok(sums / 256 + 2), ADN_ERR_INVALID,
              "adn_op_selective_scan_backward: batch too large");
    ScanParams p = params(*a, q);
    p.local = a->workspace;
    p.dsum = p.local + q.local;
    p.part_a = p.dsum + q.dsum;
    p.part_bc = p.part_a + q.part_a;
    return dispatch<kBackward>(*a, p, q.ns, static_cast<hipStream_t>(hip_stream));
}

extern "C" int adn_op_selective_scan_step(const adn_scan_args* a, void* hip_stream) {
    ADN_TRY(check(a, "adn_op_selective_scan_step", false));
    if (a->batch == 0) return ADN_OK;
    ADN_CHECK(a->steps == 1 && !a->lens, ADN_ERR_INVALID, "adn_op_selective_scan_step: one frame, no lengths");
    ADN_CHECK(a->state_out, ADN_ERR_INVALID, "adn_op_selective_scan_step: null state");
    ADN_CHECK(grid_ok((int64_t)a->batch * a->channels / 64 + 1), ADN_ERR_INVALID, "adn_op_selective_scan_step: batch * channels too large");
    const Plan q = plan_of(a->batch, 1, a->channels, a->states, a->groups, false);
    return dispatch<kStep>(*a, params(*a, q), q.ns, static_cast<hipStream_t>(hip_stream));
}
