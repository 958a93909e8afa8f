// spec_verify.cu — verification of drafted tokens (ds_cuda_tree_verify_dev,
// ds_cuda_tree_verify_greedy_dev), the target's probabilities
// (ds_cuda_token_probs_dev) and the commit of accepted K and V rows
// (ds_cuda_tree_commit_dev).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>

#include "common.cuh"
#include "ctx.h"

namespace cg = cooperative_groups;

namespace ds {

constexpr int SV_MAX_NODES = 256;
constexpr int SV_MAX_VOCAB = 1 << 18;
constexpr int SV_THREADS = 512;
constexpr int SV_WARPS = SV_THREADS / 32;
constexpr int SV_CLUSTER = 8;  // CTAs a row of the vocabulary is spread over, at most

// Every CTA of a cluster arrives when it starts and waits before it first
// writes to another's shared memory, which has to exist by then.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait_started() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A probability as a whole multiple of 2^-44, clamped to [0, 1] (NaN is 0):
// at most 2^18 of them sum to less than 2^63, whatever the order.
__device__ __forceinline__ unsigned long long sv_fixed(float p) {
    if (!(p > 0.f)) return 0;
    return (unsigned long long)__fmul_rn(fminf(p, 1.f), 0x1p44f);
}
__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(DS_FULL, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(DS_FULL, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// One cluster per sequence; its CTAs hold a row's residual r in registers,
// up to VPT values a thread: CTA k the indices from k * slice, warp w of it
// `run` consecutive ones, read 32 at a time. Every CTA walks the tree by
// itself (the walk needs single probabilities, gathered at the start, and
// the masses of the rejections at the current node); a row is read only
// where a rejection needs its residual's mass, or the next token is drawn.
// What bounds it is latency: the gather, then per row pass one read of the
// row (two with a draft) and one exchange of sums in the cluster. A chain of 7
// over 129280 tokens takes 7.8 us (5.8 with nothing to verify), 16 trees of 30
// with up to two rows and three exchanges 15.9 us, 64 trees of 15 over 32001
// tokens 15.2 us; with certain drafts 7.2, 17.5 and 10.6 us (in a graph, the
// same inputs each time). Rows read ahead of the walk make the first 10.8 us:
// most of them turn out not to be needed. VPT = 64 (more than 131072 tokens)
// spills 196 bytes.
template <int VPT>
__global__ void __launch_bounds__(SV_THREADS) tree_verify_kernel(const __grid_constant__ ds_cuda_tree_verify_t d) {
    __shared__ int par[SV_MAX_NODES], tok[SV_MAX_NODES], way[SV_MAX_NODES];
    __shared__ float acc_u[SV_MAX_NODES], pt[SV_MAX_NODES], pd[SV_MAX_NODES], mass[SV_MAX_NODES];
    __shared__ int gone[SV_MAX_NODES];
    __shared__ unsigned long long wsum[SV_WARPS], csum[2][SV_CLUSTER];
    const cg::cluster_group cl = cg::this_cluster();
    cluster_started();
    const int ncta = cl.num_blocks(), rank = cl.block_rank();
    const int b = blockIdx.x / ncta, n = d.n_nodes, V = d.vocab, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cnt = d.nodes ? min(max(d.nodes[b], 0), n) : n;
    const float *target = d.target + b * d.target_stride[0];
    const float *draft = d.draft ? d.draft + b * d.draft_stride[0] : nullptr;
    const float u_last = d.sample_u[b];
    if (tid < cnt) {
        const int p = d.parents[(size_t)b * n + tid], x = d.tokens[(size_t)b * n + tid];
        par[tid] = p;
        tok[tid] = x;
        acc_u[tid] = d.accept_u[(size_t)b * n + tid];
        const bool ok = p >= 0 && p < tid && x >= 0 && x < V;
        pt[tid] = ok ? target[p * d.target_stride[1] + x] : 0.f;
        pd[tid] = ok && draft ? draft[p * d.draft_stride[1] + x] : 1.f;
    }
    __syncthreads();
    cluster_wait_started();

    const int slice = (V + ncta - 1) / ncta, run = (slice + SV_THREADS - 1) / SV_THREADS * 32;  // run <= 32 VPT
    const int v0 = rank * slice + warp * run + lane;            // this thread's indices: v0 + 32 j
    const int vend = min(min(V, (rank + 1) * slice), rank * slice + (warp + 1) * run);
    const int jn = max(0, (vend - v0 + 31) / 32);
    float r[VPT];
    unsigned long long total = 0, below = 0;
    int parity = 0;
    // the sum over the vocabulary; leaves the warps' sums in wsum and the
    // CTAs' in csum[parity ^ 1]
    auto sum = [&]() {
        unsigned long long s = 0;
#pragma unroll
        for (int j = 0; j < VPT; j++)
            if (j < jn) s += sv_fixed(r[j]);
        s = warp_sum_u64(s);
        __syncthreads();  // the previous readers of wsum are done
        if (lane == 0) wsum[warp] = s;
        __syncthreads();
        if (tid < ncta) {
            unsigned long long c = 0;
#pragma unroll
            for (int w = 0; w < SV_WARPS; w++) c += wsum[w];
            cl.map_shared_rank(&csum[parity][0], tid)[rank] = c;
        }
        cl.sync();
        total = below = 0;
        for (int k = 0; k < ncta; k++) {
            if (k < rank) below += csum[parity][k];
            total += csum[parity][k];
        }
        parity ^= 1;
    };
    auto load = [&](const float *row) {
#pragma unroll
        for (int j = 0; j < VPT; j++)
            if (j < jn) r[j] = __ldg(row + v0 + 32 * j);
    };

    // Rejections are numbered through the whole walk, those at the current node
    // from `base` on: no entry of mass and gone is written twice, so a warp that
    // still replays an earlier node's reads what was there, and those it reads
    // have a barrier (sum's) behind them.
    int cur = 0, nrej = 0, base = 0, deep = 0;
    float m = 1.f;
    if (tid == 0) way[0] = 0;
    for (int c = 1; c < cnt; c++) {
        if (par[c] != cur) continue;
        const int x = tok[c];
        const float p = pd[c];
        float rx = pt[c];  // r(x): the rejections so far replayed for one token
        for (int k = base; k < nrej; k++)
            if (draft || gone[k] == x) rx = fmaxf(__fsub_rn(rx, __fmul_rn(mass[k], p)), 0.f);
        if (x >= 0 && x < V && __fmul_rn(acc_u[c], __fmul_rn(p, m)) < rx) {
            cur = c;
            base = nrej;
            m = 1.f;
            deep++;
            if (tid == 0) way[deep] = c;
            continue;
        }
        const float *row = target + cur * d.target_stride[1];
        if (nrej == base) load(row);
        if (draft) {
            const float *drow = draft + cur * d.draft_stride[1];
            float q[VPT];
#pragma unroll
            for (int j = 0; j < VPT; j++)
                if (j < jn) q[j] = __ldg(drow + v0 + 32 * j);
#pragma unroll
            for (int j = 0; j < VPT; j++)
                if (j < jn) r[j] = fmaxf(__fsub_rn(r[j], __fmul_rn(m, q[j])), 0.f);
        } else {
#pragma unroll
            for (int j = 0; j < VPT; j++)
                if (j < jn && v0 + 32 * j == x) r[j] = fmaxf(__fsub_rn(r[j], m), 0.f);
        }
        if (tid == 0) {
            mass[nrej] = m;
            gone[nrej] = x;
        }
        nrej++;
        sum();
        m = __fmul_rn((float)total, 0x1p-44f);
    }
    // the next token: from the residual whose sums were taken last, or from
    // the target's row where nothing was rejected or no mass is left
    if (nrej == base || total == 0) {
        load(target + cur * d.target_stride[1]);
        sum();
    }
    if (rank == 0) {
        __syncthreads();  // way is written
        for (int j = tid; j < n; j += SV_THREADS) d.path[(size_t)b * n + j] = j <= deep ? way[j] : -1;
        if (tid == 0) d.accepted[b] = deep;
        if (tid == 0 && total == 0) d.token[b] = -1;
    }
    const unsigned long long u = (unsigned long long)__fmul_rn(fminf(fmaxf(u_last, 0.f), 0x1.fffffep-1f), 0x1p24f);
    const unsigned long long lim = (total >> 24) * u + (((total & 0xffffffull) * u) >> 24);  // < total
    // the warp whose indices hold the threshold finds the 32 and the one
    for (int w = 0; w < warp; w++) below += wsum[w];
    if (lim < below || lim >= below + wsum[warp]) return;
    unsigned long long s[VPT];
#pragma unroll
    for (int j = 0; j < VPT; j++) s[j] = j < jn ? sv_fixed(r[j]) : 0;
    int j0 = 0;
    if (VPT == 64) {  // which half
        unsigned long long h = 0;
#pragma unroll
        for (int j = 0; j < 32; j++) h += s[j];
        h = warp_sum_u64(h);
        if (lim >= below + h) {
            below += h;
            j0 = 32;
#pragma unroll
            for (int j = 0; j < 32; j++) s[j] = s[VPT - 32 + j];
        }
    }
    unsigned long long own[32];
#pragma unroll
    for (int j = 0; j < 32; j++) own[j] = s[j];
    // sums over the lanes of 32 values at once: after the step of width o a
    // lane holds o values, those whose index agrees with it in the upper bits
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int k = 0; k < o; k++) {
            const unsigned long long keep = up ? s[k + o] : s[k], give = up ? s[k] : s[k + o];
            s[k] = keep + __shfl_xor_sync(DS_FULL, give, o);
        }
    }
    unsigned long long cum = warp_scan_u64(s[0]);  // lane j: the sum of the values up to j
    unsigned hit = __ballot_sync(DS_FULL, below + cum > lim);
    const int j = __ffs(hit) - 1;
    below += __shfl_sync(DS_FULL, cum - s[0], j);
    unsigned long long e = 0;
#pragma unroll
    for (int k = 0; k < 32; k++)
        if (k == j) e = own[k];
    cum = warp_scan_u64(e);
    hit = __ballot_sync(DS_FULL, below + cum > lim);
    if (lane == __ffs(hit) - 1) d.token[b] = v0 + 32 * (j0 + j);
}

// A warp per sequence, its trees in shared memory; the current node's children
// are looked for 32 nodes at a time. Bound by latency: one tree of 16
// takes 2.3 us, 64 of 64 or 256 nodes 3.1 and 3.4 us (9.2 and 30 with a thread
// per sequence).
__global__ void __launch_bounds__(32) tree_verify_greedy_kernel(const int *tokens, const int *parents, const int *nodes,
                                                                const int *want, int n, int *path, int *accepted, int *token) {
    __shared__ int par[SV_MAX_NODES], tok[SV_MAX_NODES], next[SV_MAX_NODES], way[SV_MAX_NODES];
    const int b = blockIdx.x, lane = threadIdx.x;
    const int cnt = nodes ? min(max(nodes[b], 0), n) : n;
    const size_t o = (size_t)b * n;
    for (int i = lane; i < n; i += 32) {
        par[i] = parents[o + i];
        tok[i] = tokens[o + i];
        next[i] = want[o + i];
        way[i] = -1;
    }
    __syncwarp();
    int cur = 0, deep = 0;
    if (lane == 0) way[0] = 0;
    for (int c0 = 0; c0 < cnt;) {
        const int c = c0 + lane;
        const unsigned hit = __ballot_sync(DS_FULL, c > cur && c < cnt && par[c] == cur && tok[c] == next[cur]);
        if (!hit) {
            c0 += 32;
            continue;
        }
        cur = c0 + __ffs(hit) - 1;  // (its children come later: the same 32 again)
        deep++;
        if (lane == 0) way[deep] = cur;
    }
    __syncwarp();
    for (int i = lane; i < n; i += 32) path[o + i] = way[i];
    if (lane == 0) {
        accepted[b] = deep;
        token[b] = next[cur];
    }
}

template <typename T> __device__ __forceinline__ float tp_f(T v) { return (float)v; }
template <> __device__ __forceinline__ float tp_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float tp_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// One cluster per row, its CTAs holding consecutive slices in shared memory as
// they came, so the logits are read once. A CTA takes its own maximum m and
// sum s of e = 2^((x - m) c), c = log2(e) / temperature; one exchange of
// (m, s) in the cluster gives every CTA the row's M and S, and p = e * (2^((m
// - M) c) / S): F32 logits are replaced by their e, of 16-bit ones e is taken
// twice (as F32 values in shared memory they take 47 us instead of 30).
// Bound by the memory, with eight CTAs of 128 threads and at most 28 KB an SM,
// some of them reading while others sum or write. 512 rows of 50257 logits,
// reads and writes together, in a graph on the same inputs: BF16 30 us, 5.2 TB/s;
// F32 43 us, 4.8 TB/s (BF16 on changing inputs 33.5 us, 4.6 TB/s). Twice
// the threads take 32 and 52 us (the fixed work of a thread: exchanges and
// ends), slices of 14 KB 35 us and 58 us, of 56 KB 34 and 45 us. 9 rows of
// 129280 F32 logits, mostly launch and exchange, take 6.0 us.
constexpr int TP_THREADS = 128, TP_SLICE = 28 << 10, TP_CLUSTER = 16;  // bytes of a CTA's slice, if 16 CTAs can
constexpr int TP_MOST = 56 << 10;                                      // values of a CTA
__device__ __forceinline__ float tp_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Four values from 16 or 8 bytes.
__device__ __forceinline__ float4 tp_four(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 tp_four(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 x = __half22float2(reinterpret_cast<const __half2 &>(u.x)), y = __half22float2(reinterpret_cast<const __half2 &>(u.y));
    return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ float4 tp_four(const __nv_bfloat16 *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ T tp_lowest() { return (T)-INFINITY; }
template <typename T>
__global__ void __launch_bounds__(TP_THREADS, 8) token_probs_kernel(const T *logits, int V, int64_t stride, const float *temp,
                                                                    float *out) {
    constexpr int E = 16 / sizeof(T);
    constexpr bool F32 = sizeof(T) == 4;
    extern __shared__ __align__(16) uint8_t store_raw[];
    __shared__ float sh[TP_THREADS / 32];
    __shared__ float2 ms[TP_CLUSTER];
    __shared__ unsigned long long key[TP_CLUSTER];
    __shared__ int bad[TP_CLUSTER];
    __shared__ unsigned long long best;
    T *const store = reinterpret_cast<T *>(store_raw);
    const cg::cluster_group cl = cg::this_cluster();
    cluster_started();
    constexpr int nt = TP_THREADS;
    const int ncta = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / ncta;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int slice = (V + ncta - 1) / ncta, i0 = min(V, rank * slice), len = min(V, i0 + slice) - i0;
    const T *x = logits + row * stride + i0;
    out += (size_t)row * V + i0;
    // the slice from buf on; store begins and ends with -infinity up to
    // multiples of four, and the 16-byte copies fall on 16 bytes there too
    const int head = min(len, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
    const int pad = (E - head) & (E - 1), wide = (len - head) / E, all = (pad + len + 3) & ~3;
    T *const buf = store + pad;
    for (int i = tid; i < wide; i += nt)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(buf + head + i * E)), "l"(x + head + i * E) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (tid < pad) store[tid] = tp_lowest<T>();
    if (tid < all - pad - len) buf[len + tid] = tp_lowest<T>();
    for (int i = tid; i < len - wide * E; i += nt) {
        const int k = i < head ? i : i + wide * E;
        buf[k] = x[k];
    }
    const float tt = temp ? temp[row] : 1.f, c1 = __fdiv_rn(1.44269504f, tt);
    // An infinite temperature: the least c, so that -infinity times c stays so
    // and all else is equal. Differences are taken by halves, (x / 2 - m / 2) 2 c,
    // because those of the largest logits pass F32's range.
    const float c = c1 == 0.f ? FLT_TRUE_MIN : c1, c2 = 2.f * c == INFINITY ? FLT_MAX : 2.f * c;
    auto weight = [&](float v, float half_m) { return tp_ex2(__fmaf_rn(0.5f, v, -half_m) * c2); };
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float m = -INFINITY;
#pragma unroll 4
    for (int i = 4 * tid; i < all; i += 4 * nt) {
        const float4 v = tp_four(store + i);
        m = fmaxf(m, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
    m = warp_max(m);
    if (lane == 0) sh[warp] = m;
    __syncthreads();
    cluster_wait_started();

    if (tt <= 0.f || c == INFINITY) {  // the largest logit has everything
        unsigned long long k = 0;
        bool nan = false;
        for (int i = tid; i < len; i += nt) {
            const float l = tp_f(buf[i]);
            nan |= !(l < INFINITY);
            const unsigned long long kk = argmax_key(l, i0 + i);
            if (l > -INFINITY && kk > k) k = kk;
        }
        if (tid == 0) best = 0;
        nan = __syncthreads_or(nan);
        atomicMax(&best, k);
        __syncthreads();
        if (tid < ncta) {
            cl.map_shared_rank(key, tid)[rank] = best;
            cl.map_shared_rank(bad, tid)[rank] = nan;
        }
        cl.sync();
        k = 0;
        for (int r = 0; r < ncta; r++) {
            nan |= bad[r];
            if (key[r] > k) k = key[r];
        }
        const int at = k ? (int)(0xffffffffu - (uint32_t)k) - i0 : -1;
        for (int i = tid; i < len; i += nt) out[i] = nan ? NAN : i == at ? 1.f : 0.f;
        return;
    }

    // (a slice of -infinity alone: its weights are 0)
#pragma unroll
    for (int w = 0; w < nt / 32; w++) m = fmaxf(m, sh[w]);
    m = fmaxf(m, -FLT_MAX);
    const float hm = 0.5f * m;
    float s = 0.f;
#pragma unroll 4
    for (int i = 4 * tid; i < all; i += 4 * nt) {
        float4 v = tp_four(store + i);
        v.x = weight(v.x, hm);
        v.y = weight(v.y, hm);
        v.z = weight(v.z, hm);
        v.w = weight(v.w, hm);
        if (F32) *reinterpret_cast<float4 *>(store + i) = v;
        s += (v.x + v.y) + (v.z + v.w);
    }
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) sh[warp] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int w = 0; w < nt / 32; w++) s += sh[w];
    if (tid < ncta) cl.map_shared_rank(ms, tid)[rank] = make_float2(m, s);
    cl.sync();
    const float2 part = lane < ncta ? ms[lane] : make_float2(-FLT_MAX, 0.f);
    const float M = warp_max(part.x), S = warp_sum(part.y * weight(part.x, 0.5f * M));
    const float f = S == 0.f ? 0.f : weight(m, 0.5f * M) / S;
    auto prob = [&](float v) { return (F32 ? v : weight(v, hm)) * f; };
    // four at a time between the output's 16-byte boundaries
    const int first = min(len, (int)((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / 4), quads = (len - first) / 4;
    for (int i = tid; i < len - 4 * quads; i += nt) {
        const int k = i < first ? i : i + 4 * quads;
        out[k] = prob(tp_f(buf[k]));
    }
    const bool even = ((pad + first) & 3) == 0;  // the same boundaries as in shared memory
#pragma unroll 4
    for (int i = tid; i < quads; i += nt) {
        const T *const b = buf + first + 4 * i;
        const float4 v = even ? tp_four(b) : make_float4(tp_f(b[0]), tp_f(b[1]), tp_f(b[2]), tp_f(b[3]));
        __stcs(reinterpret_cast<float4 *>(out + first + 4 * i), make_float4(prob(v.x), prob(v.y), prob(v.z), prob(v.w)));
    }
}

// A CTA per tensor, layer and sequence (and share of its rows): 16 bytes a
// thread at a time, four reads before the writes. Bound by the memory, and by
// the launch where little moves: 2.6 us for one sequence's rows in 12 layers,
// 11.8 us for 16 sequences of 6 to 43 rows (13 us with one read a thread), in a
// graph on the same rows; 5 and 14.3 us on changing ones.
constexpr int CM_THREADS = 256;
__global__ void __launch_bounds__(CM_THREADS) tree_commit_kernel(const __grid_constant__ ds_cuda_tree_commit_t d) {
    __shared__ int from[SV_MAX_NODES];
    const int chunks = d.head_dim / 8;
    const int t = blockIdx.z % d.n_tensors, l = blockIdx.z / d.n_tensors, b = blockIdx.y, tid = threadIdx.x;
    const int len = min(max(d.lens[b], 0), d.kv_max);
    const int rows = min(min(max(d.accepted[b], 0), d.n_nodes - 1) + 1, d.kv_max - len);
    if (blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) d.new_lens[b] = len + rows;
    if (tid < rows) from[tid] = d.path[(size_t)b * d.n_nodes + tid];
    __syncthreads();
    const int64_t *const cs = d.cache_stride[t], *const ts = d.tree_stride[t];
    const uint16_t *const src = (const uint16_t *)d.tree[t] + l * ts[0] + b * ts[1];
    uint16_t *const dst = (uint16_t *)d.cache[t] + l * cs[0] + b * cs[1] + len * cs[3];
    const int total = rows * d.n_kv_heads * chunks, step = gridDim.x * CM_THREADS;
    for (int i = blockIdx.x * CM_THREADS + tid; i < total; i += 4 * step) {
        uint4 v[4];
        int64_t to[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int x = i + k * step, c = x % chunks, j = x / chunks % rows, h = x / chunks / rows;
            const int f = x < total ? from[j] : -1;
            to[k] = f < 0 || f >= d.n_nodes ? -1 : h * cs[2] + j * cs[3] + 8 * c;
            if (to[k] >= 0) v[k] = __ldcs(reinterpret_cast<const uint4 *>(src + h * ts[2] + f * ts[3] + 8 * c));
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (to[k] >= 0) *reinterpret_cast<uint4 *>(dst + to[k]) = v[k];
    }
}

}  // namespace ds

using namespace ds;

static cudaStream_t sv_stream(const ds_cuda_ctx *c, void *s) { return s ? (cudaStream_t)s : c->stream; }

static cudaError_t launch_cluster(const void *f, long long ctas, int threads, size_t smem, int ncta, cudaStream_t st,
                                  void **args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ncta;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelExC(&cfg, f, args);
    if (e != cudaSuccess) cudaGetLastError();  // reported by the caller, not by whoever asks next
    return e;
}

extern "C" int ds_cuda_tree_verify_dev(ds_cuda_ctx_t *c, const ds_cuda_tree_verify_t *d, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (!d || d->batch < 0 || d->n_nodes <= 0 || d->n_nodes > SV_MAX_NODES || d->vocab <= 0 || d->vocab > SV_MAX_VOCAB)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_verify: unsupported shape batch=%d n_nodes=%d (<= %d) vocab=%d (<= %d)",
                        d ? d->batch : 0, d ? d->n_nodes : 0, SV_MAX_NODES, d ? d->vocab : 0, SV_MAX_VOCAB);
    if (d->batch == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!d->tokens || !d->parents || !d->target || !d->accept_u || !d->sample_u || !d->path || !d->accepted || !d->token)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_verify: null pointer");
    const CtxDevice on(c);
    cudaStream_t st = sv_stream(c, stream);
    // enough CTAs for the row to fit the registers; more where the batch
    // leaves SMs idle, which shortens a row's pass
    const bool wide = d->vocab > SV_CLUSTER * SV_THREADS * 32;
    int ncta = 1;
    while (ncta < SV_CLUSTER && (ncta * SV_THREADS * 32 < d->vocab ||
                                 (d->vocab > ncta * SV_THREADS && d->batch * ncta * 2 <= c->sm_count)))
        ncta *= 2;
    ds_cuda_tree_verify_t a = *d;
    void *args[] = {&a};
    return ctx_cuda(c, launch_cluster(wide ? (const void *)tree_verify_kernel<64> : (const void *)tree_verify_kernel<32>,
                                      (long long)d->batch * ncta, SV_THREADS, 0, ncta, st, args), "tree_verify launch");
}

extern "C" int ds_cuda_tree_verify_greedy_dev(ds_cuda_ctx_t *c, const int *tokens, const int *parents, const int *nodes,
                                              const int *target_tokens, int batch, int n_nodes, int *path,
                                              int *accepted, int *token, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (batch < 0 || n_nodes <= 0 || n_nodes > SV_MAX_NODES)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_verify_greedy: batch=%d n_nodes=%d (<= %d)", batch, n_nodes,
                        SV_MAX_NODES);
    if (batch == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!tokens || !parents || !target_tokens || !path || !accepted || !token)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_verify_greedy: null pointer");
    const CtxDevice on(c);
    cudaStream_t st = sv_stream(c, stream);
    tree_verify_greedy_kernel<<<batch, 32, 0, st>>>(tokens, parents, nodes, target_tokens, n_nodes, path, accepted, token);
    return ctx_cuda(c, cudaGetLastError(), "tree_verify_greedy launch");
}

extern "C" int ds_cuda_token_probs_dev(ds_cuda_ctx_t *c, int type, const void *logits, int rows, int vocab,
                                       int64_t row_stride, const float *temperature, float *probs, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (type < 0 || type > DS_CUDA_SPEC_F32 || rows < 0 || vocab <= 0)
        return ctx_fail(c, DS_CUDA_EINVAL, "token_probs: type=%d rows=%d vocab=%d", type, rows, vocab);
    if (rows == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!logits || !probs) return ctx_fail(c, DS_CUDA_EINVAL, "token_probs: null pointer");
    const CtxDevice on(c);
    cudaStream_t st = sv_stream(c, stream);
    if (vocab > TP_CLUSTER * TP_MOST)
        return ctx_fail(c, DS_CUDA_EINVAL, "token_probs: vocab %d (<= %d)", vocab, TP_CLUSTER * TP_MOST);
    // CTAs for the slices to be small; more where few rows leave SMs idle
    const int size = type == DS_CUDA_SPEC_F32 ? 4 : 2;
    int ncta = 1;
    while (ncta < TP_CLUSTER && ((vocab + ncta - 1) / ncta > TP_SLICE / size ||
                                 (vocab > ncta * 2048 && rows * ncta * 2 <= c->sm_count)))
        ncta *= 2;
    const void *f = type == DS_CUDA_SPEC_F32   ? (const void *)token_probs_kernel<float>
                    : type == DS_CUDA_SPEC_F16 ? (const void *)token_probs_kernel<__half>
                                               : (const void *)token_probs_kernel<__nv_bfloat16>;
    static std::atomic<uint64_t> ready[3];  // by type: devices (of the first 64) whose attributes are set
    if (c->device >= 64 || !(ready[type].load() >> c->device & 1)) {
        cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, TP_MOST * 4 + 64);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return ctx_cuda(c, e, "token_probs attributes");
        if (c->device < 64) ready[type].fetch_or(1ull << c->device);
    }
    void *args[] = {(void *)&logits, &vocab, &row_stride, (void *)&temperature, &probs};
    return ctx_cuda(c, launch_cluster(f, (long long)rows * ncta, TP_THREADS, (size_t)((vocab + ncta - 1) / ncta) * size + 64,
                                      ncta, st, args),
                    "token_probs launch");
}

extern "C" int ds_cuda_tree_commit_dev(ds_cuda_ctx_t *c, const ds_cuda_tree_commit_t *d, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (!d || d->n_tensors <= 0 || d->n_tensors > 8 || d->layers < 0 || d->batch < 0 || d->batch > 65535 ||
        d->n_nodes <= 0 || d->n_nodes > SV_MAX_NODES || d->n_kv_heads <= 0 || d->head_dim <= 0 || d->head_dim % 8 ||
        d->kv_max < 0 || (int64_t)d->layers * d->n_tensors > 65535 ||
        (int64_t)d->n_kv_heads * d->head_dim > INT32_MAX / SV_MAX_NODES)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_commit: unsupported shape");
    if (d->batch == 0 || d->layers == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!d->lens || !d->path || !d->accepted || !d->new_lens || d->new_lens == d->lens)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_commit: null pointer, or new_lens is lens");
    for (int t = 0; t < d->n_tensors; t++) {
        uintptr_t bits = reinterpret_cast<uintptr_t>(d->cache[t]) | reinterpret_cast<uintptr_t>(d->tree[t]);
        const int extent[4] = {d->layers, d->batch, d->n_kv_heads, d->kv_max};
        for (int k = 0; k < 4; k++) {  // the stride of a dimension of one element is never used
            if (extent[k] > 1) bits |= (uintptr_t)(2 * d->cache_stride[t][k]);
            if ((k == 3 ? d->n_nodes : extent[k]) > 1) bits |= (uintptr_t)(2 * d->tree_stride[t][k]);
        }
        if (!d->cache[t] || !d->tree[t] || bits % 16)
            return ctx_fail(c, DS_CUDA_EINVAL, "tree_commit: tensor %d: null, or base or strides not multiples of 16 bytes", t);
    }
    const CtxDevice on(c);
    cudaStream_t st = sv_stream(c, stream);
    // as many rows as could be accepted; about eight CTAs an SM
    const int work = (d->n_kv_heads * d->n_nodes * (d->head_dim / 8) + 4 * CM_THREADS - 1) / (4 * CM_THREADS);
    const long long others = (long long)d->batch * d->layers * d->n_tensors;
    const int blocks = (int)std::max<long long>(1, std::min<long long>(work, (8ll * c->sm_count + others - 1) / others));
    tree_commit_kernel<<<dim3(blocks, d->batch, d->layers * d->n_tensors), CM_THREADS, 0, st>>>(*d);
    return ctx_cuda(c, cudaGetLastError(), "tree_commit launch");
}
