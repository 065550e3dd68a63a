// Short causal convolution of every channel with its own K <= 8 taps over a (B, T, C) tensor, with bias and optional SiLU; forward,
// backward and the form for single frames.
//
//   pre[t] = bias + sum_k w[k] x[t - (K - 1) + k],  y = pre or pre sigmoid(pre)          frames before t = 0: the carried history
//   dpre = dy (sg (1 + pre (1 - sg))),  dx[t] = sum_k w[k] dpre[t + (K - 1) - k],  dw[k] = sum dpre[t] x[t - (K - 1) + k]
//
// Bound: HBM, x once and y once (backward: x, dy and dx once).  A lane owns V neighbouring channels and walks a run of time steps
// with the taps' window in registers, so a run costs K - 1 frames beyond its own (backward: K - 1 on each side, the second of them
// for the dpre behind the run's end; those come from the caches).  The backward pass adds dw and dbias in registers over all the
// runs of a workgroup, which leaves one partial row; sum_parts adds them in a fixed order.  4 x 4096 x 4096 bfloat16, 4 taps: forward
// 50 us (5.4 TB/s), backward 97 us (4.1 TB/s); 520 utterances of 12 to 40 frames x 1000: 23 and 37 us, where the one chunk of frames
// in flight per wave leaves the loads' latency in sight.
// Vectors are read at any element's address, and where V does not divide C the last lane's channels begin at C - V: it computes some of
// its neighbour's again and writes the same values.  float32, 5 taps, 373 utterances of up to 2120 frames x 105: forward 121 us, with one channel
// a lane 236; backward 288, 297.  Below 64 V channels lanes are left over (7 of 64 work at 50 channels of bfloat16).
// Frames at and behind lens[b] are padding: not read, zero in y and dx; the history left behind is that of the last valid frames.
#include "seq_common.h"

namespace adn {
namespace seq {

namespace {

struct ConvParams {
    const int32_t* lens;
    const float* w;        // [K][C]
    const float* bias;     // [C] or null
    const void* state;     // [B][K-1][C] or null (zeros)
    void* state_out;       // forward / step
    void* dstate;          // backward, or null
    float* part;           // backward: [parts][K+1][C]
    int B, T, C, K;
    int run, runs;         // time steps of a run, runs per utterance
    int parts;
    int silu;
};

// x at frame t of utterance b, channels c .. c + V: the history before 0, zero behind the length
template <typename T, int V>
__device__ __forceinline__ vec_t<T, V> frame(const View<const T>& x, const ConvParams& p, int b, int t, int c, int len) {
    if (t >= 0 && t < len) return load_raw<T, V>(x.row(b, t) + c);
    if (t < 0 && p.state) return load_raw<T, V>(static_cast<const T*>(p.state) + ((int64_t)b * (p.K - 1) + t + p.K - 1) * p.C + c);
    return vec_t<T, V>{};
}

constexpr int kConvChunk = 4;      // frames loaded together, one chunk ahead of the arithmetic

// frames t .. t + kConvChunk of x; inside the utterance without a branch per frame
template <typename T, int V>
__device__ __forceinline__ void frames(const View<const T>& x, const ConvParams& p, int b, int t, int c, int len, vec_t<T, V> (&out)[kConvChunk]) {
    if (t >= 0 && t + kConvChunk <= len) {
        const T* row = x.row(b, t) + c;
#pragma unroll
        for (int i = 0; i < kConvChunk; ++i) out[i] = load_raw<T, V>(row + i * x.st);
    } else {
#pragma unroll
        for (int i = 0; i < kConvChunk; ++i) out[i] = frame<T, V>(x, p, b, t + i, c, len);
    }
}

// workgroup: 64 lanes x V channels, 4 waves = 4 runs
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_forward_kernel(View<const T> x, View<T> y, ConvParams p) {
    const int item = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);      // B runs < 2^31 - 4
    const int own = ((int)blockIdx.y * 64 + (int)(threadIdx.x & 63)) * V, c = min(own, p.C - V);
    if (item >= p.B * p.runs || own >= p.C) return;
    const int b = item / p.runs, ri = item - b * p.runs;
    const int t0 = ri * p.run, t1 = min(p.T, t0 + p.run), len = valid_steps(p.lens, b, p.T);
    float w[K][V], bias[V];
#pragma unroll
    for (int k = 0; k < K; ++k) load_vec<float, V>(p.w + (int64_t)k * p.C + c, w[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = 0.f;
    if (p.bias) load_vec<float, V>(p.bias + c, bias);
    float win[K - 1 + kConvChunk][V];
    vec_t<T, V> next[kConvChunk];
    frames<T, V>(x, p, b, t0, c, len, next);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) widen<T, V>(frame<T, V>(x, p, b, t0 - (K - 1) + k, c, len), win[k]);
    for (int t = t0; t < t1; t += kConvChunk) {
#pragma unroll
        for (int i = 0; i < kConvChunk; ++i) widen<T, V>(next[i], win[K - 1 + i]);
        if (t + kConvChunk < t1) frames<T, V>(x, p, b, t + kConvChunk, c, len, next);
        T* row = y.row(b, t) + c;
#pragma unroll
        for (int i = 0; i < kConvChunk; ++i) {
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float a = bias[j];
#pragma unroll
                for (int k = 0; k < K; ++k) a += w[k][j] * win[i + k][j];
                if (p.silu) a *= sigmoidf(a);
                o[j] = t + i < len ? a : 0.f;
            }
            if (t + i < t1) store_vec<T, V>(row + i * y.st, o);
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) win[k][j] = win[kConvChunk + k][j];
    }
    if (ri == 0 && p.state_out) {      // the K - 1 frames before frame `len`
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
            store_raw<T, V>(static_cast<T*>(p.state_out) + ((int64_t)b * (K - 1) + k) * p.C + c, frame<T, V>(x, p, b, len - (K - 1) + k, c, len));
    }
}

// workgroup: 64 lanes x V channels, 4 waves; wave w of workgroup part q walks runs 4 q + w, + 4 parts, ...
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_backward_kernel(View<const T> x, View<const T> dy, View<T> dx, ConvParams p) {
    __shared__ float comb[4][(K + 1) * 64 * V];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int own = ((int)blockIdx.y * 64 + lane) * V, c = min(own, p.C - V);
    float dw[K + 1][V];
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) dw[k][j] = 0.f;
    if (own < p.C) {
        float w[K][V], bias[V];
#pragma unroll
        for (int k = 0; k < K; ++k) load_vec<float, V>(p.w + (int64_t)k * p.C + c, w[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) bias[j] = 0.f;
        if (p.bias) load_vec<float, V>(p.bias + c, bias);
        const int items = p.B * p.runs;                        // < 2^31 - 65536, and a step is at most 4096: no overflow
        for (int item = (int)blockIdx.x * 4 + wv; item < items; item += p.parts * 4) {
            const int b = item / p.runs, ri = item - b * p.runs;
            const int t0 = ri * p.run, t1 = min(p.T, t0 + p.run), len = valid_steps(p.lens, b, p.T);
            const auto gradients = [&](int t, vec_t<T, V> (&out)[kConvChunk]) {
                if (t + kConvChunk <= len) {
                    const T* row = dy.row(b, t) + c;
#pragma unroll
                    for (int i = 0; i < kConvChunk; ++i) out[i] = load_raw<T, V>(row + i * dy.st);
                } else {
#pragma unroll
                    for (int i = 0; i < kConvChunk; ++i) out[i] = t + i < len ? load_raw<T, V>(dy.row(b, t + i) + c) : vec_t<T, V>{};
                }
            };
            // dx of frames t0 .. t1 needs dpre of t0 .. t1 + K - 1; the history's gradient is dx at -(K-1) .. 0, the first run's
            float xw[K - 1 + kConvChunk][V], pw[K - 1 + kConvChunk][V];
            vec_t<T, V> xn[kConvChunk], gn[kConvChunk];
            frames<T, V>(x, p, b, t0, c, len, xn);
            gradients(t0, gn);
#pragma unroll
            for (int k = 0; k < K - 1; ++k) {
                widen<T, V>(frame<T, V>(x, p, b, t0 - (K - 1) + k, c, len), xw[k]);
#pragma unroll
                for (int j = 0; j < V; ++j) pw[k][j] = 0.f;
            }
            // step t brings dpre[t] and finishes dx[t - (K - 1)].  Before a run's start the window holds zeros for the dpre of earlier
            // frames: dx[t - (K - 1)] for t < t0 + K - 1 is then incomplete and belongs to the run before (or to the history).  Behind
            // the run's last frame, and behind the length, dpre adds to dx only, and behind the length it is zero
            const int stop = t1 + K - 1;
            const int sum_end = min(t1, len);       // dpre is zero behind the length, but an infinity in the window would make that NaN
            for (int t = t0; t < stop; t += kConvChunk) {
                float g[kConvChunk][V];
#pragma unroll
                for (int i = 0; i < kConvChunk; ++i) {
                    widen<T, V>(xn[i], xw[K - 1 + i]);
                    widen<T, V>(gn[i], g[i]);
                }
                if (t + kConvChunk < stop) {
                    frames<T, V>(x, p, b, t + kConvChunk, c, len, xn);
                    gradients(t + kConvChunk, gn);
                }
#pragma unroll
                for (int i = 0; i < kConvChunk; ++i) {
                    float o[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float d = g[i][j];
                        if (p.silu) {
                            float a = bias[j];
#pragma unroll
                            for (int k = 0; k < K; ++k) a += w[k][j] * xw[i + k][j];
                            const float sg = sigmoidf(a);
                            d = t + i < len ? d * (sg * (1.f + a * (1.f - sg))) : 0.f;
                        }
                        pw[K - 1 + i][j] = d;
                        float q = 0.f;
#pragma unroll
                        for (int k = 0; k < K; ++k) q += w[k][j] * pw[i + K - 1 - k][j];
                        o[j] = q;
                    }
                    const int s = t + i - (K - 1);
                    if (s >= t0 && s < t1) {
                        if (s >= len)
#pragma unroll
                            for (int j = 0; j < V; ++j) o[j] = 0.f;
                        store_vec<T, V>(dx.row(b, s) + c, o);
                    } else if (s < 0 && p.dstate)
                        store_vec<T, V>(static_cast<T*>(p.dstate) + ((int64_t)b * (K - 1) + s + K - 1) * p.C + c, o);
                    if (t + i < sum_end) {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float d = pw[K - 1 + i][j];
                            dw[K][j] += d;
#pragma unroll
                            for (int k = 0; k < K; ++k) dw[k][j] += d * xw[i + k][j];
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < K - 1; ++k)
#pragma unroll
                    for (int j = 0; j < V; ++j) { xw[k][j] = xw[kConvChunk + k][j]; pw[k][j] = pw[kConvChunk + k][j]; }
            }
        }
    }
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) comb[wv][(k * 64 + lane) * V + j] = dw[k][j];
    __syncthreads();
    float* out = p.part + (int64_t)blockIdx.x * (K + 1) * p.C;
    for (int i = threadIdx.x; i < (K + 1) * 64 * V; i += 256) {
        const int k = i / (64 * V), j = i % V, of = (int)blockIdx.y * 64 * V + i % (64 * V) - j;
        if (of < p.C) out[(int64_t)k * p.C + min(of, p.C - V) + j] = ((comb[0][i] + comb[1][i]) + comb[2][i]) + comb[3][i];
    }
}

// one frame of every utterance: y, and the history moved on by it in place
template <typename T, int V, int K>
__global__ __launch_bounds__(64) void conv_step_kernel(const T* __restrict__ x, int64_t ldx, T* __restrict__ y, int64_t ldy, ConvParams p) {
    const int c = ((int)blockIdx.x * 64 + (int)threadIdx.x) * V, b = blockIdx.y + blockIdx.z * 65535;
    if (c >= p.C || b >= p.B) return;               // (the history moves in place, so V divides C here: no channel twice)
    T* st = static_cast<T*>(p.state_out) + (int64_t)b * (K - 1) * p.C + c;
    float win[K][V], w[K][V], bias[V], o[V];
#pragma unroll
    for (int k = 0; k < K; ++k) load_vec<float, V>(p.w + (int64_t)k * p.C + c, w[k]);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load_vec<T, V>(st + (int64_t)k * p.C, win[k]);
    load_vec<T, V>(x + b * ldx + c, win[K - 1]);
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = 0.f;
    if (p.bias) load_vec<float, V>(p.bias + c, bias);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float a = bias[j];
#pragma unroll
        for (int k = 0; k < K; ++k) a += w[k][j] * win[k][j];
        if (p.silu) a *= sigmoidf(a);
        o[j] = a;
    }
    store_vec<T, V>(y + b * ldy + c, o);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store_vec<T, V>(st + (int64_t)k * p.C, win[k + 1]);
}

constexpr int kMaxTaps = 8;

int check(const adn_conv_args* a, const char* who) {
    ADN_CHECK(a, ADN_ERR_INVALID, std::string(who) + ": null arguments");
    ADN_CHECK(a->dtype == ADN_DTYPE_F32 || a->dtype == ADN_DTYPE_BF16, ADN_ERR_INVALID, std::string(who) + ": dtype is ADN_DTYPE_F32 or ADN_DTYPE_BF16");
    ADN_CHECK(a->batch >= 0 && a->steps >= 0 && (int64_t)a->batch * a->steps < ((int64_t)1 << 31) - 65536, ADN_ERR_INVALID, std::string(who) + ": bad (batch, steps)");
    ADN_CHECK(a->channels >= 1 && a->channels <= 1 << 20, ADN_ERR_INVALID, std::string(who) + ": channels outside 1 .. 2^20");
    ADN_CHECK(a->taps >= 1 && a->taps <= kMaxTaps, ADN_ERR_INVALID, std::string(who) + ": taps outside 1 .. 8");
    ADN_CHECK(a->activation == ADN_CONV_LINEAR || a->activation == ADN_CONV_SILU, ADN_ERR_INVALID, std::string(who) + ": activation is ADN_CONV_LINEAR or ADN_CONV_SILU");
    ADN_CHECK(a->weight, ADN_ERR_INVALID, std::string(who) + ": null weight");
    return ADN_OK;
}

// time steps of a run, of 64 V channels: as long as 2048 waves (two per SIMD) are left -- short runs read more frames twice -- and of
// about equal length in an utterance
int run_length(int64_t B, int64_t T, int cblocks) {
    int64_t runs = (T + 63) / 64;
    while (B * runs * cblocks < 2048 && (T + runs - 1) / runs > 8) runs *= 2;
    return (int)std::max<int64_t>((T + runs - 1) / runs, std::min<int64_t>(T, 8));
}
constexpr int kConvBwdV = 4;
// backward: workgroups along the runs; two waves per SIMD over the whole launch
int conv_parts(int64_t B, int64_t T, int C, int v, int* run) {
    const int cblocks = cdiv(C, 64 * v);
    *run = run_length(B, T, cblocks);
    const int64_t items = B * ((T + *run - 1) / *run);
    return (int)std::max<int64_t>(1, std::min<int64_t>((items + 3) / 4, cdiv(1024, cblocks)));
}
int conv_bwd_vec(const adn_conv_args& a) { return a.channels >= kConvBwdV ? kConvBwdV : 1; }

ConvParams params(const adn_conv_args& a) {
    ConvParams p{};
    p.lens = a.lens; p.w = a.weight; p.bias = a.bias; p.state = a.state; p.state_out = a.state_out; p.dstate = a.dstate;
    p.B = a.batch; p.T = a.steps; p.C = a.channels; p.K = a.taps; p.silu = a.activation == ADN_CONV_SILU;
    return p;
}

enum Pass { kForward, kBackward, kStep };

template <typename T, int V, Pass PASS, int K> int launch_k(const adn_conv_args& a, const ConvParams& p, hipStream_t s) {
    const int cblocks = cdiv(p.C, 64 * V);
    if constexpr (PASS == kForward) {
        const int64_t blocks = ((int64_t)p.B * p.runs + 3) / 4;
        hipLaunchKernelGGL((conv_forward_kernel<T, V, K>), dim3((unsigned)blocks, cblocks), dim3(256), 0, s, cview<T>(a.x), view<T>(a.y), p);
    } else if constexpr (PASS == kBackward) {
        hipLaunchKernelGGL((conv_backward_kernel<T, V, K>), dim3(p.parts, cblocks), dim3(256), 0, s, cview<T>(a.x), cview<T>(a.dy), view<T>(a.dx), p);
    } else {
        hipLaunchKernelGGL((conv_step_kernel<T, V, K>), dim3(cblocks, std::min(p.B, 65535), cdiv(p.B, 65535)), dim3(64), 0, s,
                           static_cast<const T*>(a.x.data), a.x.stride_b, static_cast<T*>(a.y.data), a.y.stride_b, p);
    }
    ADN_HIP_CHECK(hipGetLastError());
    return ADN_OK;
}
template <typename T, int V, Pass PASS> int launch(const adn_conv_args& a, const ConvParams& p, hipStream_t s) {
    switch (p.K) {
        case 1: return launch_k<T, V, PASS, 1>(a, p, s);
        case 2: return launch_k<T, V, PASS, 2>(a, p, s);
        case 3: return launch_k<T, V, PASS, 3>(a, p, s);
        case 4: return launch_k<T, V, PASS, 4>(a, p, s);
        case 5: return launch_k<T, V, PASS, 5>(a, p, s);
        case 6: return launch_k<T, V, PASS, 6>(a, p, s);
        case 7: return launch_k<T, V, PASS, 7>(a, p, s);
        default: return launch_k<T, V, PASS, 8>(a, p, s);
    }
}

}  // namespace
}  // namespace seq
}  // namespace adn

using namespace adn;
using namespace adn::seq;

extern "C" int64_t adn_op_causal_conv_workspace(int32_t batch, int32_t steps, int32_t channels, int32_t taps) {
    if (batch < 0 || steps < 0 || channels < 1 || taps < 1 || taps > kMaxTaps) return -1;
    if (batch == 0) return 0;
    steps = std::max(steps, 1);      // (no frames: the history's gradient is still written)
    int run;      // one bound for the vector and the scalar kernels
    const int parts = std::max(conv_parts(batch, steps, channels, 1, &run), conv_parts(batch, steps, channels, kConvBwdV, &run));
    return (int64_t)parts * (taps + 1) * channels;
}

extern "C" int adn_op_causal_conv_forward(const adn_conv_args* a, void* hip_stream) {
    ADN_TRY(check(a, "adn_op_causal_conv_forward"));
    const int e = a->dtype == ADN_DTYPE_BF16 ? 2 : 4;
    if (a->batch == 0) return ADN_OK;
    ADN_CHECK(a->steps == 0 || (seq_ok(a->x, e) && seq_ok(a->y, e)), ADN_ERR_INVALID, "adn_op_causal_conv_forward: null or misaligned tensor");
    ADN_CHECK(a->taps == 1 || (a->state_out && a->state_out != a->state && ptr_aligned(a->state_out, e)), ADN_ERR_INVALID,
              "adn_op_causal_conv_forward: state_out is null, misaligned or the history that is read");
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    ConvParams p = params(*a);
    const int v = a->dtype == ADN_DTYPE_BF16 ? 8 : 4;
    const bool al = a->channels >= v;
    p.run = run_length(p.B, std::max(p.T, 1), cdiv(p.C, 64 * (al ? v : 1)));
    p.runs = std::max(1, cdiv(p.T, p.run));      // (no frames: the history is still handed on)
    ADN_CHECK(grid_ok(((int64_t)p.B * p.runs + 3) / 4), ADN_ERR_INVALID, "adn_op_causal_conv_forward: batch too large");
    if (a->dtype == ADN_DTYPE_BF16) return al ? launch<__bf16, 8, kForward>(*a, p, s) : launch<__bf16, 1, kForward>(*a, p, s);
    return al ? launch<float, 4, kForward>(*a, p, s) : launch<float, 1, kForward>(*a, p, s);
}

extern "C" int adn_op_causal_conv_backward(const adn_conv_args* a, void* hip_stream) {
    ADN_TRY(check(a, "adn_op_causal_conv_backward"));
    const int e = a->dtype == ADN_DTYPE_BF16 ? 2 : 4;
    ADN_CHECK(a->dweight && a->dbias, ADN_ERR_INVALID, "adn_op_causal_conv_backward: null gradient");
    const int64_t need = adn_op_causal_conv_workspace(a->batch, a->steps, a->channels, a->taps);
    ADN_CHECK(need == 0 || (a->workspace && a->workspace_floats >= need), ADN_ERR_INVALID,
              "adn_op_causal_conv_backward: workspace smaller than adn_op_causal_conv_workspace() floats");
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    ConvParams p = params(*a);
    if (need) {
        ADN_CHECK(a->steps == 0 || (seq_ok(a->x, e) && seq_ok(a->dy, e) && seq_ok(a->dx, e)), ADN_ERR_INVALID,
                  "adn_op_causal_conv_backward: null or misaligned tensor");
        const int v = conv_bwd_vec(*a);
        p.parts = conv_parts(p.B, std::max(p.T, 1), p.C, v, &p.run);
        p.runs = std::max(1, cdiv(p.T, p.run));
        ADN_CHECK((int64_t)p.B * p.runs < ((int64_t)1 << 31) - 65536, ADN_ERR_INVALID, "adn_op_causal_conv_backward: batch too large");
        p.part = a->workspace;
        if (a->dtype == ADN_DTYPE_BF16) ADN_TRY((v == 1 ? launch<__bf16, 1, kBackward>(*a, p, s) : launch<__bf16, kConvBwdV, kBackward>(*a, p, s)));
        else ADN_TRY((v == 1 ? launch<float, 1, kBackward>(*a, p, s) : launch<float, kConvBwdV, kBackward>(*a, p, s)));
    }
    SumSegs segs{{a->dweight, a->dbias}, {(int64_t)a->taps * a->channels, a->channels}, 2};
    return sum_parts(a->workspace, (int64_t)(a->taps + 1) * a->channels, p.parts, segs, s);
}

extern "C" int adn_op_causal_conv_step(const adn_conv_args* a, void* hip_stream) {
    ADN_TRY(check(a, "adn_op_causal_conv_step"));
    const int e = a->dtype == ADN_DTYPE_BF16 ? 2 : 4;
    if (a->batch == 0) return ADN_OK;
    ADN_CHECK(a->steps == 1 && !a->lens, ADN_ERR_INVALID, "adn_op_causal_conv_step: one frame, no lengths");
    ADN_CHECK(a->batch < 65535 * 1024, ADN_ERR_INVALID, "adn_op_causal_conv_step: batch too large");
    ADN_CHECK(seq_ok(a->x, e) && seq_ok(a->y, e), ADN_ERR_INVALID, "adn_op_causal_conv_step: null or misaligned tensor");
    ADN_CHECK(a->taps == 1 || (a->state_out && ptr_aligned(a->state_out, e)), ADN_ERR_INVALID, "adn_op_causal_conv_step: null or misaligned history");
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const ConvParams p = params(*a);
    const int v = a->dtype == ADN_DTYPE_BF16 ? 8 : 4;
    const bool al = a->channels % v == 0;
    if (a->dtype == ADN_DTYPE_BF16) return al ? launch<__bf16, 8, kStep>(*a, p, s) : launch<__bf16, 1, kStep>(*a, p, s);
    return al ? launch<float, 4, kStep>(*a, p, s) : launch<float, 1, kStep>(*a, p, s);
}
