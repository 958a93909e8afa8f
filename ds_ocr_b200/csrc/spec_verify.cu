// spec_verify.cu — verification of drafted tokens (ds_cuda_tree_verify_dev,
// ds_cuda_tree_verify_greedy_dev), the target's probabilities
// (ds_cuda_token_probs_dev) and the commit of accepted K and V rows
// (ds_cuda_tree_commit_dev).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ctx.h"

namespace ds {

constexpr int SV_MAX_NODES = 256;
constexpr int SV_MAX_VOCAB = 1 << 18;
constexpr int SV_THREADS = 1024;

// A probability as a whole multiple of 2^-44, clamped to [0, 1] (NaN is 0):
// at most 2^18 of them sum to less than 2^63, whatever the order.
__device__ __forceinline__ unsigned long long sv_fixed(float p) {
    if (!(p > 0.f)) return 0;
    return (unsigned long long)__fmul_rn(fminf(p, 1.f), 0x1p44f);
}

__device__ __forceinline__ unsigned long long sv_block_sum(unsigned long long v, unsigned long long *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(DS_FULL, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < SV_THREADS / 32; w++) v += sh[w];
    return v;
}

// One CTA per sequence. r(x) is recomputed from the probabilities by
// replaying the node's rejections (their masses and tokens are kept).
__global__ void __launch_bounds__(SV_THREADS) tree_verify_kernel(const __grid_constant__ ds_cuda_tree_verify_t d) {
    __shared__ unsigned long long sh[SV_THREADS / 32];
    __shared__ float mass[SV_MAX_NODES];
    __shared__ int gone[SV_MAX_NODES];
    __shared__ unsigned long long part[SV_THREADS];
    const int b = blockIdx.x, n = d.n_nodes, V = d.vocab, tid = threadIdx.x;
    const int cnt = d.nodes ? min(max(d.nodes[b], 0), n) : n;
    const int *par = d.parents + (size_t)b * n, *tok = d.tokens + (size_t)b * n;
    int *path = d.path + (size_t)b * n;
    const float *target = d.target + b * d.target_stride[0];
    const float *draft = d.draft ? d.draft + b * d.draft_stride[0] : nullptr;
    int cur = 0, nrej = 0, deep = 0;
    float m = 1.f;
    auto resid = [&](int x) {
        float r = target[cur * d.target_stride[1] + x];
        if (draft) {
            const float p = draft[cur * d.draft_stride[1] + x];
            for (int k = 0; k < nrej; k++) r = fmaxf(__fsub_rn(r, __fmul_rn(mass[k], p)), 0.f);
        } else {
            for (int k = 0; k < nrej; k++)
                if (gone[k] == x) r = fmaxf(__fsub_rn(r, mass[k]), 0.f);
        }
        return r;
    };
    if (tid == 0) path[0] = 0;
    for (int c = 1; c < cnt; c++) {
        if (par[c] != cur) continue;
        const int x = tok[c];
        bool ok = false;
        if (x >= 0 && x < V) {
            const float p = draft ? draft[cur * d.draft_stride[1] + x] : 1.f;
            ok = __fmul_rn(d.accept_u[(size_t)b * n + c], __fmul_rn(p, m)) < resid(x);
        }
        if (ok) {
            cur = c;
            nrej = 0;
            m = 1.f;
            deep++;
            if (tid == 0) path[deep] = c;
        } else {
            __syncthreads();
            if (tid == 0) {
                mass[nrej] = m;
                gone[nrej] = x;
            }
            __syncthreads();
            nrej++;
            unsigned long long s = 0;
            for (int v = tid; v < V; v += SV_THREADS) s += sv_fixed(resid(v));
            m = __fmul_rn((float)sv_block_sum(s, sh), 0x1p-44f);
        }
    }
    for (int j = deep + 1 + tid; j < n; j += SV_THREADS) path[j] = -1;
    // the next token: each thread's run of V, then the run that holds the threshold
    const int run = (V + SV_THREADS - 1) / SV_THREADS, v0 = min(V, tid * run), v1 = min(V, v0 + run);
    unsigned long long total = 0;
    for (int pass = 0; pass < 2 && total == 0; pass++) {
        if (pass) nrej = 0;
        unsigned long long s = 0;
        for (int v = v0; v < v1; v++) s += sv_fixed(resid(v));
        total = sv_block_sum(s, sh);
        part[tid] = s;
    }
    __syncthreads();
    if (tid) return;
    int t = -1;
    if (total) {
        const unsigned long long u = (unsigned long long)__fmul_rn(fminf(fmaxf(d.sample_u[b], 0.f), 0x1.fffffep-1f), 0x1p24f);
        const unsigned long long lim = (total >> 24) * u + (((total & 0xffffffull) * u) >> 24);
        unsigned long long cum = 0;
        int k = 0;
        while (k < SV_THREADS - 1 && cum + part[k] <= lim) cum += part[k++];
        for (t = k * run; t < V - 1; t++) {
            cum += sv_fixed(resid(t));
            if (cum > lim) break;
        }
    }
    d.token[b] = t;
    d.accepted[b] = deep;
}

__global__ void tree_verify_greedy_kernel(const int *tokens, const int *parents, const int *nodes, const int *want,
                                          int batch, int n, int *path, int *accepted, int *token) {
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= batch) return;
    const int cnt = nodes ? min(max(nodes[b], 0), n) : n;
    const size_t o = (size_t)b * n;
    int cur = 0, deep = 0;
    path[o] = 0;
    for (int c = 1; c < cnt; c++)
        if (parents[o + c] == cur && tokens[o + c] == want[o + cur]) {
            cur = c;
            path[o + ++deep] = c;
        }
    for (int j = deep + 1; j < n; j++) path[o + j] = -1;
    accepted[b] = deep;
    token[b] = want[o + cur];
}

template <typename T> __device__ __forceinline__ float tp_f(T v) { return (float)v; }
template <> __device__ __forceinline__ float tp_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float tp_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// One CTA per row, three passes.
template <typename T>
__global__ void __launch_bounds__(1024) token_probs_kernel(const T *logits, int V, int64_t stride, const float *temp, float *out) {
    __shared__ float sh[32];
    __shared__ unsigned long long best;
    const T *x = logits + blockIdx.x * stride;
    out += (size_t)blockIdx.x * V;
    const float tt = temp ? temp[blockIdx.x] : 1.f;
    const int tid = threadIdx.x;
    float m = -INFINITY;
    bool bad = false;
    unsigned long long key = 0;
    for (int v = tid; v < V; v += 1024) {
        const float l = tp_f(x[v]);
        bad |= isnan(l);
        m = fmaxf(m, l);
        const unsigned long long k = argmax_key(l, v);
        if (!isnan(l) && k > key) key = k;
    }
    if (tid == 0) best = 0;
    bad = __syncthreads_or(bad);
    atomicMax(&best, key);
    m = warp_max(m);
    if ((tid & 31) == 0) sh[tid >> 5] = m;
    __syncthreads();
    for (int w = 0; w < 32; w++) m = fmaxf(m, sh[w]);
    __syncthreads();
    if (bad || m == INFINITY || isnan(tt)) {
        for (int v = tid; v < V; v += 1024) out[v] = NAN;
        return;
    }
    if (m == -INFINITY || tt <= 0.f) {
        const int at = m == -INFINITY ? -1 : (int)(0xffffffffu - (uint32_t)best);
        for (int v = tid; v < V; v += 1024) out[v] = v == at ? 1.f : 0.f;
        return;
    }
    float s = 0.f;
    for (int v = tid; v < V; v += 1024) s += expf((tp_f(x[v]) - m) / tt);
    s = warp_sum(s);
    if ((tid & 31) == 0) sh[tid >> 5] = s;
    __syncthreads();
    s = 0.f;
    for (int w = 0; w < 32; w++) s += sh[w];
    for (int v = tid; v < V; v += 1024) out[v] = expf((tp_f(x[v]) - m) / tt) / s;
}

// One thread per 16 bytes of a row.
__global__ void tree_commit_kernel(const __grid_constant__ ds_cuda_tree_commit_t d) {
    const int chunks = d.head_dim / 8;
    const int t = blockIdx.z % d.n_tensors, l = blockIdx.z / d.n_tensors, b = blockIdx.y;
    const int len = min(max(d.lens[b], 0), d.kv_max);
    const int rows = min(min(max(d.accepted[b], 0), d.n_nodes - 1) + 1, d.kv_max - len);
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) d.new_lens[b] = len + rows;
    for (int64_t i = blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)rows * d.n_kv_heads * chunks;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int c = i % chunks, h = (i / chunks) % d.n_kv_heads, j = i / chunks / d.n_kv_heads;
        const int src = d.path[(size_t)b * d.n_nodes + j];
        if (src < 0 || src >= d.n_nodes) continue;
        const int64_t *cs = d.cache_stride[t], *ts = d.tree_stride[t];
        const uint16_t *from = (const uint16_t *)d.tree[t] + l * ts[0] + b * ts[1] + h * ts[2] + src * ts[3] + 8 * c;
        uint16_t *to = (uint16_t *)d.cache[t] + l * cs[0] + b * cs[1] + h * cs[2] + (len + j) * cs[3] + 8 * c;
        *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(from);
    }
}

}  // namespace ds

using namespace ds;

static cudaStream_t sv_stream(ds_cuda_ctx *c, void *s) {
    cudaSetDevice(c->device);
    return s ? (cudaStream_t)s : c->stream;
}

extern "C" int ds_cuda_tree_verify_dev(ds_cuda_ctx_t *c, const ds_cuda_tree_verify_t *d, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (!d || d->batch < 0 || d->n_nodes <= 0 || d->n_nodes > SV_MAX_NODES || d->vocab <= 0 || d->vocab > SV_MAX_VOCAB)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_verify: unsupported shape batch=%d n_nodes=%d (<= %d) vocab=%d (<= %d)",
                        d ? d->batch : 0, d ? d->n_nodes : 0, SV_MAX_NODES, d ? d->vocab : 0, SV_MAX_VOCAB);
    if (d->batch == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!d->tokens || !d->parents || !d->target || !d->accept_u || !d->sample_u || !d->path || !d->accepted || !d->token)
        return ctx_fail(c, DS_CUDA_EINVAL, "tree_verify: null pointer");
    cudaStream_t st = sv_stream(c, stream);
    tree_verify_kernel<<<d->batch, SV_THREADS, 0, st>>>(*d);
    return ctx_cuda(c, cudaGetLastError(), "tree_verify launch");
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
    cudaStream_t st = sv_stream(c, stream);
    tree_verify_greedy_kernel<<<(batch + 31) / 32, 32, 0, st>>>(tokens, parents, nodes, target_tokens, batch, n_nodes,
                                                                path, accepted, token);
    return ctx_cuda(c, cudaGetLastError(), "tree_verify_greedy launch");
}

extern "C" int ds_cuda_token_probs_dev(ds_cuda_ctx_t *c, int type, const void *logits, int rows, int vocab,
                                       int64_t row_stride, const float *temperature, float *probs, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (type < 0 || type > DS_CUDA_SPEC_F32 || rows < 0 || vocab <= 0)
        return ctx_fail(c, DS_CUDA_EINVAL, "token_probs: type=%d rows=%d vocab=%d", type, rows, vocab);
    if (rows == 0) return DS_CUDA_OK;  // an empty tensor has no address
    if (!logits || !probs) return ctx_fail(c, DS_CUDA_EINVAL, "token_probs: null pointer");
    cudaStream_t st = sv_stream(c, stream);
    if (type == DS_CUDA_SPEC_F32)
        token_probs_kernel<<<rows, 1024, 0, st>>>((const float *)logits, vocab, row_stride, temperature, probs);
    else if (type == DS_CUDA_SPEC_F16)
        token_probs_kernel<<<rows, 1024, 0, st>>>((const __half *)logits, vocab, row_stride, temperature, probs);
    else
        token_probs_kernel<<<rows, 1024, 0, st>>>((const __nv_bfloat16 *)logits, vocab, row_stride, temperature, probs);
    return ctx_cuda(c, cudaGetLastError(), "token_probs launch");
}

extern "C" int ds_cuda_tree_commit_dev(ds_cuda_ctx_t *c, const ds_cuda_tree_commit_t *d, void *stream) {
    if (!c || !c->ok) return DS_CUDA_EINVAL;
    if (!d || d->n_tensors <= 0 || d->n_tensors > 8 || d->layers < 0 || d->batch < 0 || d->batch > 65535 ||
        d->n_nodes <= 0 || d->n_nodes > SV_MAX_NODES || d->n_kv_heads <= 0 || d->head_dim <= 0 || d->head_dim % 8 ||
        d->kv_max < 0 || (int64_t)d->layers * d->n_tensors > 65535)
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
    cudaStream_t st = sv_stream(c, stream);
    const int blocks = (d->n_kv_heads * d->n_nodes * (d->head_dim / 8) + 255) / 256;
    tree_commit_kernel<<<dim3(blocks < 8 ? blocks : 8, d->batch, d->layers * d->n_tensors), 256, 0, st>>>(*d);
    return ctx_cuda(c, cudaGetLastError(), "tree_commit launch");
}
