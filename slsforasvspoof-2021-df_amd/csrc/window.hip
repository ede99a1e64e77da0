// Attention with a sliding window and a few first tokens that stay visible, for recordings of any length: forward and
// backward.
//
//   visible(i, j) = j < len and j <= i + right and (j >= i - left or j < sinks),   i < len
//   S = scale Q K^T on visible pairs, P = softmax(S) by rows, O = P V, lse = log sum exp S
//   dV = P^T dO,  dS = P o (dO V^T - rowsum(dO o O)),  dQ = scale dS K,  dK = scale dS^T Q
// Query head h reads key head h / (Hq / Hk).  A row with nothing visible (a padded frame) yields 0, lse = -inf and no gradient.
//
// Products run on the 32 x 32 x 16 MFMA, scores TRANSPOSED (keys on the row index, S^T = K Q^T): a lane then holds one
// query and four consecutive keys per register group, so row statistics need one exchange between the halves of the wave,
// and the packed probabilities ARE the B operand of O^T = V^T P^T when the 16 keys of a step are enumerated as
// (half hi, j) -> 4 hi + j (j < 4), 8 + 4 hi + j - 4: P never leaves registers.  V^T comes from row-major LDS by
// ds_read_b64_tr_b16.  The key loop visits only the tiles of the sinks and of the window.
#include "kernels.h"
#include "window.h"

namespace slsmi {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct HeadPtr {
    const bf16_t* p;
    long b, r, h;   // element strides of batch, row, head
};
struct HeadOut {
    bf16_t* p;
    long b, r, h;
};

struct WinArgs {
    HeadPtr q, k, v, o, d;   // o, d (dO): backward
    HeadOut out, dq, dk, dv;
    float* lse;              // [B][Hq][T]
    float* delta;            // [B][Hq][T]: rowsum(dO o O), written by the dQ kernel
    float* part;             // sink keys' partial sums (see window_dkv_kernel)
    const int* nframes;
    int B, T, Hq, Hk;
    int left, right, sinks;  // left, right in [0, T]; sinks in [0, SINK_MAX]
    int tiles;               // tiles of a head in this launch
    int far_blocks, far_chunk;   // dkv: workgroups per sink block beyond the near tiles, queries per workgroup
    float scale;
};

constexpr int SINK_MAX = 128;

// LDS image of a tile of rows of D 16-bit values, without padding: 16-byte chunks of a row permuted by its row number so
// that 16 consecutive rows read at one chunk (ds_read_b128 of the row operand) and four consecutive rows read at four
// neighbouring chunks (ds_read_b64_tr_b16 of the transposed operand) both touch every bank once.
template <int D>
__device__ __forceinline__ int tile_at(int row, int chunk) {
    if constexpr (D == 64) return row * 128 + ((chunk ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3))) << 4);
    else return row * 256 + ((chunk ^ (((row & 3) << 2) | ((row >> 2) & 3))) << 4);
}

template <int D>
__device__ __forceinline__ u16x8 row_frag(const char* tile, int row, int chunk) {
    return *reinterpret_cast<const u16x8*>(tile + tile_at<D>(row, chunk));
}

// A operand of the transposed product for column block dt (32 columns) and the 16 rows row0 ..: rows enumerated as above
template <int D>
__device__ __forceinline__ u16x8 tr_frag(const char* tile, int row0, int dt, int lane) {
    const int row = row0 + ((lane >> 5) << 2) + ((lane & 15) >> 2);
    const int col = dt * 32 + (lane & 16) + (lane & 3) * 4;
    const int in = (col & 4) * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(tile + tile_at<D>(row, col >> 3) + in));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(tile + tile_at<D>(row + 8, col >> 3) + in));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Rows row0 .. row0 + ROWS - 1 of a head on their way to LDS: requested early, written when the tile before is used up.
// Rows at or past `len` become zeros (what lies there may be anything, NaN among it).
template <int D, int ROWS>
struct Stage {
    static constexpr int CH = D / 8;
    static constexpr int N = ROWS * CH / 256;
    u16x8 v[N];
    __device__ __forceinline__ void load(const bf16_t* head, long rs, int row0, int len, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * 256, row = row0 + c / CH;
            v[i] = *reinterpret_cast<const u16x8*>(head + (long)min(row, len - 1) * rs + (c & (CH - 1)) * 8);
            if (row >= len) v[i] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        }
    }
    __device__ __forceinline__ void store(char* tile, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * 256;
            *reinterpret_cast<u16x8*>(tile + tile_at<D>(c / CH, c & (CH - 1))) = v[i];
        }
    }
};

// Workgroup number -> (batch x head, tile): consecutive workgroups go to the 8 XCDs in turn, and each XCD gets a
// contiguous share of the work, so that the tiles of a head -- which read the same keys -- meet in one L2.
__device__ __forceinline__ unsigned xcd_order(unsigned n, unsigned total) {
    const unsigned x = n & 7, i = n >> 3, q = total >> 3, r = total & 7;
    return x * q + (x < r ? x : r) + i;
}

// Whether the 32 keys k0 .. and the 32 queries q0 .. have visible pairs, and whether all pairs are.
struct Vis {
    bool any, all;
};
__device__ __forceinline__ Vis block_visibility(int q0, int k0, int len, int left, int right, int sinks) {
    Vis r;
    r.any = k0 < len && q0 < len && k0 <= q0 + 31 + right && (k0 + 31 >= q0 - left || k0 < sinks);
    r.all = k0 + 31 < len && k0 + 31 <= q0 + right && (k0 >= q0 + 31 - left || k0 + 31 < sinks);
    return r;
}

// The key tiles (of BN) that queries qa .. qb see: [0, st) of the sinks, then [w0, w0 + n - st)
struct KeyTiles {
    int st, w0, n;
    __device__ __forceinline__ int tile(int i) const { return i < st ? i : w0 + i - st; }
};
__device__ __forceinline__ KeyTiles key_tiles(int qa, int qb, int len, int left, int right, int sinks, int BN) {
    const int lo = max(qa - left, 0), hi = min(qb + right, len - 1);
    KeyTiles t;
    t.w0 = lo / BN;
    t.st = min((sinks + BN - 1) / BN, t.w0);
    t.n = t.st + hi / BN - t.w0 + 1;
    return t;
}

// 32 x 32 tile of a transposed result (row = 8 (r / 4) + 4 hi + r % 4, column = lane % 32), rows dt * 32 .. of D: the
// halves of the wave exchange so that each lane stores 16 contiguous bytes of its column's row of memory.
template <int FMT, bool UNIT>
__device__ __forceinline__ void store_column(bf16_t* dst, int dt, f32x16 v, int hi) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[8 * p + 2 * i], b = v[8 * p + 2 * i + 1];
            w[i] = UNIT ? Op<FMT>::pack2_unit(a, b) : Op<FMT>::pack2(a, b);
        }
        const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        *reinterpret_cast<u32x4*>(dst + dt * 32 + p * 16 + hi * 8) = u32x4{x[0], y[0], x[1], y[1]};
    }
}

template <int FMT>
__device__ __forceinline__ u16x8 pack_step(const f32x16& p, int s) {
    return __builtin_bit_cast(u16x8, u32x4{Op<FMT>::pack2(p[8 * s], p[8 * s + 1]), Op<FMT>::pack2(p[8 * s + 2], p[8 * s + 3]),
                                           Op<FMT>::pack2(p[8 * s + 4], p[8 * s + 5]), Op<FMT>::pack2(p[8 * s + 6], p[8 * s + 7])});
}
template <int FMT>
__device__ __forceinline__ u16x8 pack_step_unit(const f32x16& p, int s) {
    return __builtin_bit_cast(u16x8, u32x4{Op<FMT>::pack2_unit(p[8 * s], p[8 * s + 1]), Op<FMT>::pack2_unit(p[8 * s + 2], p[8 * s + 3]),
                                           Op<FMT>::pack2_unit(p[8 * s + 4], p[8 * s + 5]), Op<FMT>::pack2_unit(p[8 * s + 6], p[8 * s + 7])});
}

__device__ __forceinline__ f32x16 zero16() {
    return f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

__device__ __forceinline__ int frames_of(const WinArgs& a, int b) { return a.nframes ? min(max(a.nframes[b], 0), a.T) : a.T; }

// ---- forward: 128 queries per workgroup, 32 per wave; 64-key tiles
template <int FMT, int D>
__global__ __launch_bounds__(256) void window_fwd_kernel(WinArgs a) {
    constexpr int BN = 64, NS = D / 16, DT = D / 32;
    __shared__ __attribute__((aligned(16))) char lds[2 * BN * D * 2];
    char* const Ks = lds;
    char* const Vs = lds + BN * D * 2;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned w = xcd_order(blockIdx.x, gridDim.x);
    const int tile = a.tiles - 1 - (int)(w % a.tiles);   // the tiles with the longest key ranges first
    const int bh = w / a.tiles, b = bh / a.Hq, h = bh % a.Hq, hk = h / (a.Hq / a.Hk);
    const int len = frames_of(a, b);
    const int q0 = tile * 128, qw = q0 + wave * 32, q = qw + col;
    bf16_t* const orow = a.out.p + b * a.out.b + h * a.out.h + (long)q * a.out.r;
    float* const lse = a.lse ? a.lse + (long)bh * a.T + q : nullptr;
    if (q0 >= len) {
        if (q < a.T) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) store_column<FMT, true>(orow, dt, zero16(), hi);
            if (lse && hi == 0) *lse = -INFINITY;
        }
        return;
    }
    const bf16_t* kh = a.k.p + b * a.k.b + hk * a.k.h;
    const bf16_t* vh = a.v.p + b * a.v.b + hk * a.v.h;
    u16x8 qf[NS];
    {
        const bf16_t* qr = a.q.p + b * a.q.b + h * a.q.h + (long)min(q, len - 1) * a.q.r + hi * 8;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const u16x8*>(qr + s * 16);
    }
    const KeyTiles kt = key_tiles(q0, min(q0 + 127, len - 1), len, a.left, a.right, a.sinks, BN);
    const float sc = a.scale * LOG2E;
    float m = -INFINITY, l = 0.f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = zero16();
    Stage<D, BN> sk, sv;
    sk.load(kh, a.k.r, kt.tile(0) * BN, len, tid);
    sv.load(vh, a.v.r, kt.tile(0) * BN, len, tid);
    for (int it = 0; it < kt.n; ++it) {
        const int k0 = kt.tile(it) * BN;
        __syncthreads();
        sk.store(Ks, tid);
        sv.store(Vs, tid);
        __syncthreads();
        if (it + 1 < kt.n) {
            sk.load(kh, a.k.r, kt.tile(it + 1) * BN, len, tid);
            sv.load(vh, a.v.r, kt.tile(it + 1) * BN, len, tid);
        }
        Vis vis[2];
        f32x16 s[2];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            vis[u] = block_visibility(qw, k0 + 32 * u, len, a.left, a.right, a.sinks);
            if (!vis[u].any) continue;
            s[u] = zero16();
#pragma unroll
            for (int e = 0; e < NS; ++e) s[u] = mfma32<FMT>(row_frag<D>(Ks, 32 * u + col, 2 * e + hi), qf[e], s[u]);
            if (!vis[u].all) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = k0 + 32 * u + 8 * (r >> 2) + 4 * hi + (r & 3);
                    const bool ok = key < len && key <= q + a.right && (key >= q - a.left || key < a.sinks);
                    s[u][r] = ok ? s[u][r] : -INFINITY;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
        }
        if (!vis[0].any && !vis[1].any) continue;
        mx = fmaxf(mx, other_half(mx)) * sc;
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        const float corr = __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (!vis[u].any) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], sc, -ref));
                sum += s[u][r];
            }
        }
        l = l * corr + sum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] *= corr;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (!vis[u].any) continue;
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const u16x8 p = pack_step_unit<FMT>(s[u], st);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] = mfma32<FMT>(tr_frag<D>(Vs, 32 * u + 16 * st, dt, lane), p, o[dt]);
            }
        }
    }
    l += other_half(l);
    const bool live = q < len;
    const float inv = live ? 1.0f / l : 0.f;
    if (q < a.T) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            f32x16 v = live ? o[dt] * inv : zero16();
            store_column<FMT, true>(orow, dt, v, hi);
        }
        if (lse && hi == 0) *lse = live ? (m + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
    }
}

// ---- backward, queries: dQ and delta = rowsum(dO o O); the forward's loop with P recomputed from lse
template <int FMT, int D>
__global__ __launch_bounds__(256) void window_dq_kernel(WinArgs a) {
    constexpr int BN = 64, NS = D / 16, DT = D / 32;
    __shared__ __attribute__((aligned(16))) char lds[2 * BN * D * 2];
    char* const Ks = lds;
    char* const Vs = lds + BN * D * 2;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned w = xcd_order(blockIdx.x, gridDim.x);
    const int tile = a.tiles - 1 - (int)(w % a.tiles);
    const int bh = w / a.tiles, b = bh / a.Hq, h = bh % a.Hq, hk = h / (a.Hq / a.Hk);
    const int len = frames_of(a, b);
    const int q0 = tile * 128, qw = q0 + wave * 32, q = qw + col;
    bf16_t* const dqrow = a.dq.p + b * a.dq.b + h * a.dq.h + (long)q * a.dq.r;
    float* const drow = a.delta + (long)bh * a.T + q;
    if (q0 >= len) {
        if (q < a.T) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) store_column<FMT, true>(dqrow, dt, zero16(), hi);
            if (hi == 0) *drow = 0.f;
        }
        return;
    }
    const bf16_t* kh = a.k.p + b * a.k.b + hk * a.k.h;
    const bf16_t* vh = a.v.p + b * a.v.b + hk * a.v.h;
    u16x8 qf[NS], df[NS];
    float delta = 0.f;
    {
        const int row = min(q, len - 1);
        const bf16_t* qr = a.q.p + b * a.q.b + h * a.q.h + (long)row * a.q.r + hi * 8;
        const bf16_t* dr = a.d.p + b * a.d.b + h * a.d.h + (long)row * a.d.r + hi * 8;
        const bf16_t* pr = a.o.p + b * a.o.b + h * a.o.h + (long)row * a.o.r + hi * 8;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            qf[s] = *reinterpret_cast<const u16x8*>(qr + s * 16);
            df[s] = *reinterpret_cast<const u16x8*>(dr + s * 16);
            const u16x8 of = *reinterpret_cast<const u16x8*>(pr + s * 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf(Op<FMT>::unpack(df[s][e]), Op<FMT>::unpack(of[e]), delta);
        }
        delta += other_half(delta);
    }
    const bool live = q < len;
    if (q < a.T && hi == 0) *drow = live ? delta : 0.f;
    const float sc = a.scale * LOG2E;
    const float ls = a.lse[(long)bh * a.T + min(q, len - 1)] * LOG2E;
    const KeyTiles kt = key_tiles(q0, min(q0 + 127, len - 1), len, a.left, a.right, a.sinks, BN);
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();
    Stage<D, BN> sk, sv;
    sk.load(kh, a.k.r, kt.tile(0) * BN, len, tid);
    sv.load(vh, a.v.r, kt.tile(0) * BN, len, tid);
    for (int it = 0; it < kt.n; ++it) {
        const int k0 = kt.tile(it) * BN;
        __syncthreads();
        sk.store(Ks, tid);
        sv.store(Vs, tid);
        __syncthreads();
        if (it + 1 < kt.n) {
            sk.load(kh, a.k.r, kt.tile(it + 1) * BN, len, tid);
            sv.load(vh, a.v.r, kt.tile(it + 1) * BN, len, tid);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const Vis vis = block_visibility(qw, k0 + 32 * u, len, a.left, a.right, a.sinks);
            if (!vis.any) continue;
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int e = 0; e < NS; ++e) {
                s = mfma32<FMT>(row_frag<D>(Ks, 32 * u + col, 2 * e + hi), qf[e], s);
                dp = mfma32<FMT>(row_frag<D>(Vs, 32 * u + col, 2 * e + hi), df[e], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[r], sc, -ls));
                const int key = k0 + 32 * u + 8 * (r >> 2) + 4 * hi + (r & 3);
                const bool ok = vis.all || (key < len && key <= q + a.right && (key >= q - a.left || key < a.sinks));
                s[r] = ok ? p * (dp[r] - delta) : 0.f;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const u16x8 e = pack_step<FMT>(s, st);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma32<FMT>(tr_frag<D>(Ks, 32 * u + 16 * st, dt, lane), e, acc[dt]);
            }
        }
    }
    if (q < a.T) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const f32x16 v = live ? acc[dt] * a.scale : zero16();
            store_column<FMT, false>(dqrow, dt, v, hi);
        }
    }
}

// ---- backward, keys: dK and dV.  A workgroup owns 128 keys (32 per wave) and goes through the 64-query tiles of every
// query head of the group that see them; S = Q K^T this time (queries on the row index), so P and dS are the B operands
// of dV^T = dO^T P and dK^T = Q^T dS.
//
// The sinks' keys are seen by every later query: the queries past the near ones of a sink block (32 keys) are cut into
// chunks of far_chunk, one workgroup each, whose four waves share the block's keys and take 32 of 128 queries in turn.
// Those sums, and the near workgroup's for sink rows, go as fp32 to `part` [B][Hk][sink block][1 + 4 far_blocks][dK, dV]
// [32 keys][D] and are added in that order by window_sink_kernel.
template <int FMT, int D>
__global__ __launch_bounds__(256, 1) void window_dkv_kernel(WinArgs a) {
    constexpr int NS = D / 16, DT = D / 32, BQ = 128;
    __shared__ __attribute__((aligned(16))) char lds[2 * BQ * D * 2];
    __shared__ __attribute__((aligned(16))) float st_l[BQ], st_d[BQ];
    char* const Qs = lds;
    char* const Ds = lds + BQ * D * 2;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sink_blocks = (a.sinks + 31) / 32;
    const int per_head = a.tiles + sink_blocks * a.far_blocks;
    const unsigned w = xcd_order(blockIdx.x, gridDim.x);
    const int bh = w / per_head, item = w % per_head, b = bh / a.Hk, hk = bh % a.Hk;
    const int len = frames_of(a, b);
    const int grp = a.Hq / a.Hk;
    const bool far = item >= a.tiles;
    int k0w, qa, qb;   // this wave's keys; queries qa .. qb
    int block = 0, chunk = 0;
    if (!far) {
        const int k0 = item * 128;
        k0w = k0 + wave * 32;
        qa = max(k0 - a.right, 0);
        qb = min(k0 + 127 + a.left, len - 1);
    } else {
        block = (item - a.tiles) / a.far_blocks;
        chunk = (item - a.tiles) % a.far_blocks;
        k0w = block * 32;
        // the near workgroup of these keys ended at this query
        const int first = (k0w / 128) * 128 + 127 + a.left + 1;
        qa = min(first + chunk * a.far_chunk, len);
        qb = min(first + (chunk + 1) * a.far_chunk, len) - 1;
    }
    const int key = k0w + col;
    u16x8 kf[NS], vf[NS];
    {
        const int row = min(key, max(len - 1, 0));
        const bf16_t* kr = a.k.p + b * a.k.b + hk * a.k.h + (long)row * a.k.r + hi * 8;
        const bf16_t* vr = a.v.p + b * a.v.b + hk * a.v.h + (long)row * a.v.r + hi * 8;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            kf[s] = *reinterpret_cast<const u16x8*>(kr + s * 16);
            vf[s] = *reinterpret_cast<const u16x8*>(vr + s * 16);
        }
    }
    f32x16 ak[DT], av[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) ak[dt] = av[dt] = zero16();
    const float sc = a.scale * LOG2E;
    const int t0 = qa / BQ, nt = (!far && item * 128 >= len) || qb < qa ? 0 : qb / BQ - t0 + 1;
    const int total = nt * grp;
    Stage<D, BQ> sq, sd;
    float l1 = 0.f, d1 = 0.f;
    auto request = [&](int it) {
        const int h = hk * grp + it / nt, q0 = (t0 + it % nt) * BQ;
        sq.load(a.q.p + b * a.q.b + h * a.q.h, a.q.r, q0, len, tid);
        sd.load(a.d.p + b * a.d.b + h * a.d.h, a.d.r, q0, len, tid);
        if (tid < BQ) {
            const long at = ((long)b * a.Hq + h) * a.T + min(q0 + tid, len - 1);
            l1 = a.lse[at] * LOG2E;
            d1 = a.delta[at];
        }
    };
    if (total > 0) request(0);
    for (int it = 0; it < total; ++it) {
        const int q0 = (t0 + it % nt) * BQ;
        __syncthreads();
        sq.store(Qs, tid);
        sd.store(Ds, tid);
        if (tid < BQ) {
            st_l[tid] = l1;
            st_d[tid] = d1;
        }
        __syncthreads();
        if (it + 1 < total) request(it + 1);
#pragma unroll 1
        for (int u = 0; u < BQ / 32; ++u) {
            if (far && u != wave) continue;
            const int qs = q0 + 32 * u;
            Vis vis = block_visibility(qs, k0w, len, a.left, a.right, a.sinks);
            if (qs > qb || qs + 31 < qa) vis.any = false;
            if (!vis.any) continue;
            const bool whole = vis.all && qs + 31 < len && qs >= qa && qs + 31 <= qb;
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int e = 0; e < NS; ++e) {
                s = mfma32<FMT>(row_frag<D>(Qs, 32 * u + col, 2 * e + hi), kf[e], s);
                dp = mfma32<FMT>(row_frag<D>(Ds, 32 * u + col, 2 * e + hi), vf[e], dp);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(st_l + 32 * u + 8 * g + 4 * hi);
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(st_d + 32 * u + 8 * g + 4 * hi);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 4 * g + j, q = qs + 8 * g + 4 * hi + j;
                    const bool ok = whole || (q >= qa && q <= qb && key < len && key <= q + a.right &&
                                              (key >= q - a.left || key < a.sinks));
                    const float p = ok ? __builtin_amdgcn_exp2f(fmaf(s[r], sc, -l4[j])) : 0.f;
                    s[r] = p;
                    dp[r] = ok ? p * (dp[r] - d4[j]) : 0.f;
                }
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const u16x8 pf = pack_step_unit<FMT>(s, st), ef = pack_step<FMT>(dp, st);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    av[dt] = mfma32<FMT>(tr_frag<D>(Ds, 32 * u + 16 * st, dt, lane), pf, av[dt]);
                    ak[dt] = mfma32<FMT>(tr_frag<D>(Qs, 32 * u + 16 * st, dt, lane), ef, ak[dt]);
                }
            }
        }
    }
    if (far || (k0w < a.sinks && a.far_blocks > 0)) {
        const int blk = far ? block : k0w / 32, slot = far ? 1 + chunk * 4 + wave : 0;
        float* dst = a.part + ((((long)bh * sink_blocks + blk) * (1 + 4 * a.far_blocks) + slot) * 2 * 32 + col) * D + 4 * hi;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 x, y;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[j] = ak[dt][4 * g + j] * a.scale;
                    y[j] = av[dt][4 * g + j];
                }
                *reinterpret_cast<f32x4*>(dst + dt * 32 + 8 * g) = x;
                *reinterpret_cast<f32x4*>(dst + 32 * D + dt * 32 + 8 * g) = y;
            }
        return;
    }
    if (key < a.T) {
        bf16_t* const dk = a.dk.p + b * a.dk.b + hk * a.dk.h + (long)key * a.dk.r;
        bf16_t* const dv = a.dv.p + b * a.dv.b + hk * a.dv.h + (long)key * a.dv.r;
        const bool live = key < len;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            store_column<FMT, false>(dk, dt, live ? ak[dt] * a.scale : zero16(), hi);
            store_column<FMT, false>(dv, dt, live ? av[dt] : zero16(), hi);
        }
    }
}

// the partial sums of a sink block (32 keys) in slot order -> its rows of dK and dV; one workgroup per (block, head, 8 keys)
template <int FMT, int D>
__global__ __launch_bounds__(256) void window_sink_kernel(WinArgs a) {
    const int sink_blocks = (a.sinks + 31) / 32, slots = 1 + 4 * a.far_blocks;
    const int kq = blockIdx.x & 3, n = blockIdx.x >> 2, blk = n % sink_blocks, bh = n / sink_blocks, b = bh / a.Hk, hk = bh % a.Hk;
    const int len = frames_of(a, b);
    for (int i = threadIdx.x; i < 2 * 8 * D / 4; i += 256) {
        const int which = i / (8 * D / 4), at = i % (8 * D / 4), kl = kq * 8 + at / (D / 4), c = (at % (D / 4)) * 4;
        const int key = blk * 32 + kl;
        if (key >= a.T) continue;
        const float* src = a.part + (((long)n * slots * 2 + which) * 32 + kl) * D + c;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        if (key < len)
            for (int j = 0; j < slots; ++j) s += *reinterpret_cast<const f32x4*>(src + (long)j * 2 * 32 * D);
        const HeadOut& d = which ? a.dv : a.dk;
        typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
        *reinterpret_cast<u32x2_t*>(d.p + b * d.b + hk * d.h + (long)key * d.r + c) =
            u32x2_t{Op<FMT>::pack2(s[0], s[1]), Op<FMT>::pack2(s[2], s[3])};
    }
}

constexpr int FAR_CHUNK = 1024;

// queries past the near ones of the first sink block, in chunks (0: none)
int far_blocks_of(int T, int left, int sinks) {
    if (sinks <= 0) return 0;
    const long first = 127L + left + 1;
    return first >= T ? 0 : (int)((T - first + FAR_CHUNK - 1) / FAR_CHUNK);
}

bool head_ok(const WindowHeads& x, int heads, int T, int D) {
    if (!x.p || ((uintptr_t)x.p & 15) || x.batch % 8 || x.row % 8 || x.head % 8) return false;
    if (x.batch < 0 || x.row < 0 || x.head < 0 || x.row > (1L << 31) || x.head > (1L << 40) || x.batch > (1L << 50)) return false;
    // rows and heads are distinct pieces of D values
    if (T > 1 && x.row < D) return false;
    if (heads > 1 && x.head < D) return false;
    return true;
}

// the ranges every call has to keep; clamps the window
bool window_args(const WindowParams& p, WinArgs& a) {
    if (p.B < 0 || p.T < 0 || p.T > (1 << 29) || p.Hk < 1 || p.Hq < p.Hk || p.Hq % p.Hk || p.Hq > 4096) return false;
    if (p.D != 64 && p.D != 128) return false;
    if (p.fmt != FMT_BF16 && p.fmt != FMT_F16) return false;
    if (!(p.scale > 0.f) || p.left < -1 || p.right < -1 || p.sinks < 0 || p.sinks > SINK_MAX) return false;
    if ((long)p.B * p.Hq * ((p.T + 127L) / 128 + 4) > 0x7fffffffL / 8) return false;
    a.B = p.B; a.T = p.T; a.Hq = p.Hq; a.Hk = p.Hk;
    a.left = p.left < 0 || p.left > p.T ? p.T : p.left;
    a.right = p.right < 0 || p.right > p.T ? p.T : p.right;
    a.sinks = a.left >= p.T ? 0 : (p.sinks < p.T ? p.sinks : p.T);
    a.scale = p.scale;
    a.nframes = p.nframes;
    a.tiles = (p.T + 127) / 128;
    return true;
}

HeadPtr in_head(const WindowHeads& x) { return {x.p, x.batch, x.row, x.head}; }
HeadOut out_head(const WindowHeads& x) { return {const_cast<bf16_t*>(x.p), x.batch, x.row, x.head}; }

size_t delta_bytes(const WinArgs& a) { return ((size_t)a.B * a.Hq * a.T * sizeof(float) + 255) & ~(size_t)255; }

}  // namespace

hipError_t launch_window_attention(const WindowParams& p, float* lse, hipStream_t s) {
    WinArgs a{};
    if (!window_args(p, a)) return hipErrorInvalidValue;
    if (p.B == 0 || p.T == 0) return hipSuccess;
    if (!head_ok(p.q, p.Hq, p.T, p.D) || !head_ok(p.k, p.Hk, p.T, p.D) || !head_ok(p.v, p.Hk, p.T, p.D) ||
        !head_ok(p.o, p.Hq, p.T, p.D))
        return hipErrorInvalidValue;
    a.q = in_head(p.q); a.k = in_head(p.k); a.v = in_head(p.v); a.out = out_head(p.o);
    a.lse = lse;
    const dim3 grid((unsigned)(p.B * p.Hq * a.tiles));
    SLSMI_FMT_DISPATCH(p.fmt, {
        if (p.D == 64) hipLaunchKernelGGL((window_fwd_kernel<F, 64>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((window_fwd_kernel<F, 128>), grid, dim3(256), 0, s, a);
    });
    return hipGetLastError();
}

size_t window_attention_bwd_workspace(const WindowParams& p) {
    WinArgs a{};
    if (!window_args(p, a) || p.B == 0 || p.T == 0) return 0;
    const size_t fb = far_blocks_of(p.T, a.left, a.sinks), sb = (a.sinks + 31) / 32;
    return delta_bytes(a) + (fb ? (size_t)p.B * p.Hk * sb * (1 + 4 * fb) * 2 * 32 * p.D * sizeof(float) : 0);
}

hipError_t launch_window_attention_bwd(const WindowParams& p, const float* lse, const WindowHeads& dout, const WindowHeads& dq,
                                       const WindowHeads& dk, const WindowHeads& dv, void* ws, size_t ws_bytes, hipStream_t s) {
    WinArgs a{};
    if (!window_args(p, a)) return hipErrorInvalidValue;
    if (p.B == 0 || p.T == 0) return hipSuccess;
    if (!head_ok(p.q, p.Hq, p.T, p.D) || !head_ok(p.k, p.Hk, p.T, p.D) || !head_ok(p.v, p.Hk, p.T, p.D) ||
        !head_ok(p.o, p.Hq, p.T, p.D) || !head_ok(dout, p.Hq, p.T, p.D) || !head_ok(dq, p.Hq, p.T, p.D) ||
        !head_ok(dk, p.Hk, p.T, p.D) || !head_ok(dv, p.Hk, p.T, p.D) || !lse)
        return hipErrorInvalidValue;
    if (!ws || ((uintptr_t)ws & 15) || ws_bytes < window_attention_bwd_workspace(p)) return hipErrorOutOfMemory;
    a.q = in_head(p.q); a.k = in_head(p.k); a.v = in_head(p.v); a.o = in_head(p.o); a.d = in_head(dout);
    a.dq = out_head(dq); a.dk = out_head(dk); a.dv = out_head(dv);
    a.lse = const_cast<float*>(lse);
    a.delta = reinterpret_cast<float*>(ws);
    a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + delta_bytes(a));
    a.far_chunk = FAR_CHUNK;
    a.far_blocks = far_blocks_of(p.T, a.left, a.sinks);
    const int sb = (a.sinks + 31) / 32;
    const dim3 gq((unsigned)(p.B * p.Hq * a.tiles)), gk((unsigned)(p.B * p.Hk * (a.tiles + sb * a.far_blocks)));
    SLSMI_FMT_DISPATCH(p.fmt, {
        if (p.D == 64) {
            hipLaunchKernelGGL((window_dq_kernel<F, 64>), gq, dim3(256), 0, s, a);
            hipLaunchKernelGGL((window_dkv_kernel<F, 64>), gk, dim3(256), 0, s, a);
        } else {
            hipLaunchKernelGGL((window_dq_kernel<F, 128>), gq, dim3(256), 0, s, a);
            hipLaunchKernelGGL((window_dkv_kernel<F, 128>), gk, dim3(256), 0, s, a);
        }
        if (a.far_blocks > 0) {
            if (p.D == 64) hipLaunchKernelGGL((window_sink_kernel<F, 64>), dim3(p.B * p.Hk * sb * 4), dim3(256), 0, s, a);
            else hipLaunchKernelGGL((window_sink_kernel<F, 128>), dim3(p.B * p.Hk * sb * 4), dim3(256), 0, s, a);
        }
    });
    return hipGetLastError();
}

}  // namespace slsmi
