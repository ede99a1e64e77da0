// One new frame per stream against a rolling cache (slsmi_window_attention_step), and the cache's prefill.
//
// Cache: k, v [B][Hk][slots][D], slots = sinks + window.  Position p lives in slot p for p < sinks, else in slot
// sinks + (p - sinks) mod window: the new frame overwrites the one that has just left the window, and slots
// 0 .. min(p + 1, slots) - 1 are exactly the frames that position p sees (the sinks and the last `window` ones).
// Softmax does not care about their order, so the kernel needs no mask beyond a count.
//
// Bound by reading the cache once (4 D bytes per slot and key head).  A wave reads 64 / (D / 8) slots at a time, 16 bytes
// per lane; the D / 8 lanes of a slot sum the products of their channels by lane moves inside a row of 16, every slot
// group keeps its own running maximum and sum, and groups, waves and the workgroups that share a long axis are joined at
// the end.  Queries stay in 32 bits (normalised and turned here, never rounded).
#include "kernels.h"
#include "window.h"

namespace slsmi {

namespace {

constexpr int ST_WAVES = 4;
constexpr int MAX_SPLITS = 128;   // workgroups that share a (stream, key head)
constexpr int MIN_SLOTS = 128;    // per workgroup, where an axis is shared
constexpr float LOG2E = 1.4426950408889634f;

struct StepArgs {
    const bf16_t* qkv;     // [B] rows of (Hq + 2 Hk) heads
    long ld;
    bf16_t* kc;
    bf16_t* vc;
    const long long* positions;   // [B]; negative: no frame for this stream
    bf16_t* out;           // [B][Hq][D]
    const float* wq;       // null: q and k come normalised and turned already
    const float* wk;
    const double* freqs;
    float* ml;             // [B][Hq][splits][2]: maximum and sum of a share
    float* acc;            // [B][Hq][splits][D]: its weighted values
    float eps, scale;
    int half, interleaved;
    int Hq, Hk, slots, sinks;
    int qblocks;           // workgroups per key head: ceil(group / GP)
    int splits, per_split; // slots per workgroup
};

template <int FMT, int D, int GP>
__global__ __launch_bounds__(ST_WAVES * 64) void window_step_kernel(StepArgs a) {
    constexpr int GL = D / 8, KG = 64 / GL, U = 4;
    __shared__ float2 tab[ST_WAVES][64];
    __shared__ float red_m[ST_WAVES][GP], red_l[ST_WAVES][GP];
    __shared__ float red_o[ST_WAVES][GP][D];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & (GL - 1), kg = lane / GL;
    const int split = blockIdx.x, hk = blockIdx.y / a.qblocks, qb = blockIdx.y % a.qblocks, b = blockIdx.z;
    const int grp = a.Hq / a.Hk;
    const int g0 = qb * GP;   // first query head of this workgroup within the group
    const long long pos = a.positions[b];
    const int s0 = split * a.per_split, s1 = min(s0 + a.per_split, a.slots);
    const int n = pos < 0 ? 0 : (int)min(pos + 1, (long long)a.slots);
    const long share = ((long)b * a.Hq + hk * grp + g0) * a.splits + split;
    if (s0 >= n) {   // nothing here (also: no frame for this stream)
        if (a.splits == 1) {
            for (int i = tid; i < GP * D; i += ST_WAVES * 64)
                if (g0 + i / D < grp) a.out[((long)b * a.Hq + hk * grp + g0) * D + i] = 0;
        } else if (tid < GP && g0 + tid < grp) {
            *reinterpret_cast<f32x2*>(a.ml + (share + (long)tid * a.splits) * 2) = f32x2{-INFINITY, 0.f};
        }
        return;
    }
    const int slot = pos < a.sinks ? (int)pos : a.sinks + (int)((pos - a.sinks) % (a.slots - a.sinks));
    const bf16_t* row = a.qkv + (long)b * a.ld + c * 8;

    // ---- the queries, and the new key and value where this workgroup owns their slot
    float q[GP][8];
    const bool own = slot >= s0 && slot < s1;
    u16x8 nk, nv;
    {
        u16x8 xq[GP];
#pragma unroll
        for (int i = 0; i < GP; ++i)
            xq[i] = *reinterpret_cast<const u16x8*>(row + (long)(hk * grp + min(g0 + i, grp - 1)) * D);
        nk = *reinterpret_cast<const u16x8*>(row + (long)(a.Hq + hk) * D);
        nv = *reinterpret_cast<const u16x8*>(row + (long)(a.Hq + a.Hk + hk) * D);
        const float sc = a.scale * LOG2E;
        if (a.wq) {
            const NormLane t = norm_lane<D>(lane, pos, norm_freq(lane, a.freqs, a.half), a.half, a.interleaved, tab[wave]);
            const int pc = t.partner & (GL - 1);
            float w[8], pw[8], y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = a.wq[c * 8 + e];
                pw[e] = a.wq[pc * 8 + e];
            }
#pragma unroll
            for (int i = 0; i < GP; ++i) {
                norm_rope_lane<FMT, D>(xq[i], w, pw, t, a.eps, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) q[i][e] = y[e] * sc;
            }
            if (own) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = a.wk[c * 8 + e];
                    pw[e] = a.wk[pc * 8 + e];
                }
                norm_rope_lane<FMT, D>(nk, w, pw, t, a.eps, y);
                u32x4 r;
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = result2<FMT>(y[2 * i], y[2 * i + 1]);
                nk = __builtin_bit_cast(u16x8, r);
            }
        } else {
#pragma unroll
            for (int i = 0; i < GP; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) q[i][e] = Op<FMT>::unpack(xq[i][e]) * sc;
        }
    }
    const long head = ((long)b * a.Hk + hk) * a.slots;
    if (own && qb == 0 && wave == 0 && kg == 0) {
        *reinterpret_cast<u16x8*>(a.kc + (head + slot) * D + c * 8) = nk;
        *reinterpret_cast<u16x8*>(a.vc + (head + slot) * D + c * 8) = nv;
    }

    // ---- the slots of this workgroup.  The slot just written is taken from registers: another wave's store need not have
    // landed yet.
    const int end = min(s1, n);
    float m[GP], l[GP], o[GP][8];
#pragma unroll
    for (int i = 0; i < GP; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[i][e] = 0.f;
    }
    const bf16_t* kb = a.kc + head * D + c * 8;
    const bf16_t* vb = a.vc + head * D + c * 8;
    for (int k0 = s0 + wave * KG * U; k0 < end; k0 += ST_WAVES * KG * U) {
        u16x8 kr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = min(k0 + u * KG + kg, end - 1);
            kr[u] = *reinterpret_cast<const u16x8*>(kb + (long)key * D);
            vr[u] = *reinterpret_cast<const u16x8*>(vb + (long)key * D);
        }
        float s[U][GP];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = k0 + u * KG + kg;
            if (own && min(key, end - 1) == slot) {   // (lanes past the end hold the last slot: finite for their zero weight)
                kr[u] = nk;
                vr[u] = nv;
            }
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = Op<FMT>::unpack(kr[u][e]);
#pragma unroll
            for (int i = 0; i < GP; ++i) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) d = fmaf(f[e], q[i][e], d);
                d = lane_group_sum<GL>(d);
                s[u][i] = key < end ? d : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < GP; ++i) {
            float mx = m[i];
#pragma unroll
            for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][i]);
            const float ref = mx == -INFINITY ? 0.f : mx;
            const float corr = __builtin_amdgcn_exp2f(m[i] - ref);
            m[i] = mx;
            l[i] *= corr;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[i][e] *= corr;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u][i] = __builtin_amdgcn_exp2f(s[u][i] - ref);
                l[i] += s[u][i];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = Op<FMT>::unpack(vr[u][e]);
#pragma unroll
            for (int i = 0; i < GP; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) o[i][e] = fmaf(s[u][i], f[e], o[i][e]);
        }
    }
    // ---- join the slot groups of the wave, then the waves
#pragma unroll
    for (int i = 0; i < GP; ++i) {
        float mx = m[i];
#pragma unroll
        for (int x = GL; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
        const float corr = __builtin_amdgcn_exp2f(m[i] - (mx == -INFINITY ? 0.f : mx));
        l[i] *= corr;
#pragma unroll
        for (int x = GL; x < 64; x <<= 1) l[i] += __shfl_xor(l[i], x, 64);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[i][e] *= corr;
#pragma unroll
            for (int x = GL; x < 64; x <<= 1) o[i][e] += __shfl_xor(o[i][e], x, 64);
        }
        if (kg == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) red_o[wave][i][c * 8 + e] = o[i][e];
            if (c == 0) {
                red_m[wave][i] = mx;
                red_l[wave][i] = l[i];
            }
        }
    }
    __syncthreads();
    for (int t = tid; t < GP * D; t += ST_WAVES * 64) {
        const int i = t / D, d = t % D;
        if (g0 + i >= grp) break;
        float mx = red_m[0][i];
#pragma unroll
        for (int w = 1; w < ST_WAVES; ++w) mx = fmaxf(mx, red_m[w][i]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < ST_WAVES; ++w) {
            const float corr = __builtin_amdgcn_exp2f(red_m[w][i] - ref);
            sum = fmaf(red_l[w][i], corr, sum);
            acc = fmaf(red_o[w][i][d], corr, acc);
        }
        if (a.splits == 1) {
            a.out[((long)b * a.Hq + hk * grp + g0 + i) * D + d] = (bf16_t)result2<FMT>(acc / sum, 0.f);
        } else {
            a.acc[(share + (long)i * a.splits) * D + d] = acc;
            if (d == 0) *reinterpret_cast<f32x2*>(a.ml + (share + (long)i * a.splits) * 2) = f32x2{mx, sum};
        }
    }
}

// Joins the shares of one query head: a wave forms the shares' weights, then D / 4 threads times 1024 / D groups of shares
// (every (1024 / D)th, in order) sum the values, and the groups are added in their order.
template <int FMT, int D>
__global__ __launch_bounds__(256) void window_step_join_kernel(const float* __restrict__ ml, const float* __restrict__ acc,
                                                               bf16_t* __restrict__ out, int splits) {
    constexpr int G = 1024 / D, C = D / 4;
    __shared__ float wt[MAX_SPLITS];
    __shared__ float total;
    __shared__ f32x4 red[G][C];
    const int tid = threadIdx.x;
    if (tid < 64) {
        float mx = -INFINITY, m[MAX_SPLITS / 64], l[MAX_SPLITS / 64];
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 64; ++i) {
            const int s = tid + 64 * i;
            const f32x2 v = s < splits ? *reinterpret_cast<const f32x2*>(ml + ((long)blockIdx.x * splits + s) * 2) : f32x2{-INFINITY, 0.f};
            m[i] = v[0];
            l[i] = v[1];
            mx = fmaxf(mx, m[i]);
        }
        mx = wave_max(mx);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 64; ++i) {
            const float w = __builtin_amdgcn_exp2f(m[i] - (mx == -INFINITY ? 0.f : mx));
            sum = fmaf(l[i], w, sum);
            wt[tid + 64 * i] = l[i] == 0.f ? 0.f : w;   // an empty share: its values were not written
        }
        sum = wave_sum(sum);
        if (tid == 0) total = sum;
    }
    __syncthreads();
    const int c = tid % C, g = tid / C;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = g; i < splits; i += G) {
        const float w = wt[i];
        if (w != 0.f) s += w * *reinterpret_cast<const f32x4*>(acc + ((long)blockIdx.x * splits + i) * D + c * 4);
    }
    red[g][c] = s;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int i = 1; i < G; ++i) s += red[i][c];
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
    *reinterpret_cast<u32x2_t*>(out + (long)blockIdx.x * D + c * 4) =
        u32x2_t{result2<FMT>(s[0] * inv, s[1] * inv), result2<FMT>(s[2] * inv, s[3] * inv)};
}

// k, v [B][T] heads -> the slots their newest positions live in; slots without a position keep what they hold
struct FillArgs {
    const bf16_t* k;
    const bf16_t* v;
    long kb, kr, kh, vb, vr, vh;
    bf16_t* kc;
    bf16_t* vc;
    const int* nframes;
    int T, Hk, D, slots, sinks;
};
__global__ __launch_bounds__(256) void window_fill_kernel(FillArgs a) {
    const int gl = a.D / 8, hk = blockIdx.y, b = blockIdx.z;
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int slot = i / gl, c = i % gl;
    const int len = a.nframes ? min(max(a.nframes[b], 0), a.T) : a.T;
    if (slot >= a.slots) return;
    int pos = slot;
    if (slot >= a.sinks) {
        const int ring = a.slots - a.sinks, last = len - 1;
        if (last < slot) return;   // the first round of the ring has not come this far
        pos = last - (last - slot) % ring;
    }
    if (pos >= len) return;
    const long dst = (((long)b * a.Hk + hk) * a.slots + slot) * a.D + c * 8;
    *reinterpret_cast<u16x8*>(a.kc + dst) = *reinterpret_cast<const u16x8*>(a.k + b * a.kb + hk * a.kh + (long)pos * a.kr + c * 8);
    *reinterpret_cast<u16x8*>(a.vc + dst) = *reinterpret_cast<const u16x8*>(a.v + b * a.vb + hk * a.vh + (long)pos * a.vr + c * 8);
}

// How many workgroups share a (stream, key head).  The join is a launch of its own: up to 512 slots of 64 channels (or the
// same bytes) one workgroup is faster alone (one stream, 16 heads x 64, graph replay: 5.0 against 6.6 us at 512 slots, 10.1
// against 6.7 at 2048).  Beyond that, enough to give every CU two, none with fewer than 128 slots.
int step_splits(int B, int heads, int slots, int D) {
    if ((long)slots * D <= 512 * 64) return 1;
    const long have = (long)B * heads, want = (512 + have - 1) / have, most = (slots + MIN_SLOTS - 1) / MIN_SLOTS;
    const long n = want < most ? want : most;
    return (int)(n < MAX_SPLITS ? n : MAX_SPLITS);
}

// query heads a workgroup serves at once
int step_heads(int grp) { return grp >= 8 ? 8 : grp >= 4 ? (grp > 4 ? 8 : 4) : grp > 2 ? 4 : grp; }

bool step_ok(const WindowStepParams& p) {
    if (p.B < 0 || p.B > 65535 || p.Hk < 1 || p.Hq < p.Hk || p.Hq % p.Hk || p.Hq > 4096) return false;
    if (p.D != 64 && p.D != 128) return false;
    if (p.sinks < 0 || p.slots <= p.sinks || p.slots > (1 << 24)) return false;
    if (p.fmt != FMT_BF16 && p.fmt != FMT_F16) return false;
    return true;
}

int step_qblocks(const WindowStepParams& p) {
    const int grp = p.Hq / p.Hk, gp = step_heads(grp);
    return (grp + gp - 1) / gp;
}

template <int FMT, int D>
void launch_step_one(int gp, dim3 grid, hipStream_t s, const StepArgs& a) {
    switch (gp) {
        case 1: hipLaunchKernelGGL((window_step_kernel<FMT, D, 1>), grid, dim3(ST_WAVES * 64), 0, s, a); break;
        case 2: hipLaunchKernelGGL((window_step_kernel<FMT, D, 2>), grid, dim3(ST_WAVES * 64), 0, s, a); break;
        case 4: hipLaunchKernelGGL((window_step_kernel<FMT, D, 4>), grid, dim3(ST_WAVES * 64), 0, s, a); break;
        default: hipLaunchKernelGGL((window_step_kernel<FMT, D, 8>), grid, dim3(ST_WAVES * 64), 0, s, a); break;
    }
}

}  // namespace

static size_t step_ml_bytes(const WindowStepParams& p, int splits) {
    return ((size_t)p.B * p.Hq * splits * 2 * sizeof(float) + 15) & ~(size_t)15;
}

size_t window_step_workspace(const WindowStepParams& p) {
    if (!step_ok(p) || p.B == 0) return 0;
    const int splits = step_splits(p.B, p.Hk * step_qblocks(p), p.slots, p.D);
    return splits > 1 ? step_ml_bytes(p, splits) + (size_t)p.B * p.Hq * splits * p.D * sizeof(float) : 0;
}

hipError_t launch_window_step(const WindowStepParams& p, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!step_ok(p)) return hipErrorInvalidValue;
    if (p.B == 0) return hipSuccess;
    auto al = [](const void* x) { return x && ((uintptr_t)x & 15) == 0; };
    if (!al(p.qkv) || !al(p.k_cache) || !al(p.v_cache) || !p.positions || !al(p.out) || p.ld % 8) return hipErrorInvalidValue;
    if (p.B > 1 && p.ld < (long)(p.Hq + 2 * p.Hk) * p.D) return hipErrorInvalidValue;
    if ((p.wq == nullptr) != (p.wk == nullptr) || (p.wq && !eps_ok(p.eps)) || !scale_ok(p.scale)) return hipErrorInvalidValue;
    if (p.half < 0 || 2 * p.half > p.D || p.half % 8 || (p.half > 0 && (!p.freqs || !p.wq))) return hipErrorInvalidValue;
    StepArgs a{};
    a.qkv = p.qkv; a.ld = p.ld; a.kc = p.k_cache; a.vc = p.v_cache; a.positions = p.positions; a.out = p.out;
    a.wq = p.wq; a.wk = p.wk; a.freqs = p.freqs; a.eps = p.eps; a.scale = p.scale; a.half = p.half;
    a.interleaved = p.interleaved; a.Hq = p.Hq; a.Hk = p.Hk; a.slots = p.slots; a.sinks = p.sinks;
    a.qblocks = step_qblocks(p);
    a.splits = step_splits(p.B, p.Hk * a.qblocks, p.slots, p.D);
    a.per_split = ((p.slots + a.splits - 1) / a.splits + 31) / 32 * 32;
    a.ml = reinterpret_cast<float*>(ws);
    a.acc = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + step_ml_bytes(p, a.splits));
    if (a.splits > 1 && (!al(ws) || ws_bytes < window_step_workspace(p))) return hipErrorOutOfMemory;
    const int gp = step_heads(p.Hq / p.Hk);
    const dim3 grid(a.splits, p.Hk * a.qblocks, p.B);
    SLSMI_FMT_DISPATCH(p.fmt, {
        if (p.D == 64) launch_step_one<F, 64>(gp, grid, s, a);
        else launch_step_one<F, 128>(gp, grid, s, a);
        if (a.splits > 1) {
            if (p.D == 64) hipLaunchKernelGGL((window_step_join_kernel<F, 64>), dim3(p.B * p.Hq), dim3(256), 0, s, a.ml, a.acc, a.out, a.splits);
            else hipLaunchKernelGGL((window_step_join_kernel<F, 128>), dim3(p.B * p.Hq), dim3(256), 0, s, a.ml, a.acc, a.out, a.splits);
        }
    });
    return hipGetLastError();
}

hipError_t launch_window_fill(const WindowHeads& k, const WindowHeads& v, bf16_t* kc, bf16_t* vc, const int* nframes, int B, int T,
                              int Hk, int D, int slots, int sinks, hipStream_t s) {
    if (B < 0 || B > 65535 || T < 0 || T > (1 << 29) || Hk < 1 || Hk > 4096 || (D != 64 && D != 128) || sinks < 0 ||
        slots <= sinks || slots > (1 << 24))
        return hipErrorInvalidValue;
    if (B == 0 || T == 0) return hipSuccess;
    auto al = [](const void* x) { return x && ((uintptr_t)x & 15) == 0; };
    if (!al(k.p) || !al(v.p) || !al(kc) || !al(vc)) return hipErrorInvalidValue;
    if (k.batch % 8 || k.row % 8 || k.head % 8 || v.batch % 8 || v.row % 8 || v.head % 8) return hipErrorInvalidValue;
    FillArgs a{k.p, v.p, k.batch, k.row, k.head, v.batch, v.row, v.head, kc, vc, nframes, T, Hk, D, slots, sinks};
    const long items = (long)slots * (D / 8);
    hipLaunchKernelGGL(window_fill_kernel, dim3((unsigned)((items + 255) / 256), Hk, B), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace slsmi
