// One token of the gated delta rule for every row of a decoding batch, state in place:
//     u = b (v - a S^T k),   S <- a S + k u^T,   o = scale S^T q = scale (a S_old^T q + (k.q) u).
// Both products with the old state come out of one reading of it, so the state is read once and written once and everything
// is in 32 bits.  A CTA takes 32 columns of one head's state (columns do not interact), held in registers in between.
// Bound by memory latency (27 % of an SM's warps resident; 72 registers a thread instead of 96 changed nothing): a batch of 96 rows, some
// padding, 16 heads of 128 x 128 moves 175 MB in 35.8 us, 4.9 TB/s (0.76 of the measured copy rate); one row of 10 heads 6 us.
#include "delta_common.cuh"

namespace dism {
namespace {

constexpr int STEP_THREADS = 128, STEP_COLUMNS = 32, STEP_GROUPS = STEP_THREADS / 8;  // eight lanes of four columns to a state row

template <int D>
__global__ void __launch_bounds__(STEP_THREADS) delta_step_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k,
                                                                  const __nv_bfloat16* __restrict__ v, const void* __restrict__ g,
                                                                  const void* __restrict__ beta, bool gates_bf16, float scale,
                                                                  float* __restrict__ state, const int* __restrict__ slots, int64_t pool,
                                                                  int batch, int key_heads, int heads, int dv,
                                                                  __nv_bfloat16* __restrict__ out) {
    constexpr int ROWS = D / STEP_GROUPS;
    __shared__ float4 part[STEP_THREADS / 32][2][8];
    __shared__ float part_kq[STEP_THREADS / 32];
    __shared__ int next_of[STEP_THREADS / 32];
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31, head = blockIdx.y;
    const int column = blockIdx.x * STEP_COLUMNS + (lane & 7) * 4, group = thread >> 3;
    const int key_head = head / (heads / key_heads);
    int row = blockIdx.z;
    const int64_t slot = slots ? __ldg(slots + row) : row;
    if (slot < 0 || slot >= pool) {  // a row without a sequence
        if (thread < 8) *reinterpret_cast<uint2*>(out + (int64_t(row) * heads + head) * dv + column) = make_uint2(0, 0);
        return;
    }
    float4* at = reinterpret_cast<float4*>(state + ((slot * heads + head) * D + group) * dv + column);
    const int64_t stride = int64_t(STEP_GROUPS) * dv / 4;
    float4 s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) s[i] = at[i * stride];
    if (slots) {  // rows that name one slot are tokens of one sequence, in order: the first row's CTAs take them all
        bool earlier = false;
        for (int i = thread; i < row; i += STEP_THREADS) earlier |= __ldg(slots + i) == slot;
        if (__syncthreads_or(earlier)) return;
    }
    for (;;) {
        const __nv_bfloat16 *qr = q + (int64_t(row) * key_heads + key_head) * D, *kr = k + (int64_t(row) * key_heads + key_head) * D;
        const float decay = expf(gate(g, int64_t(row) * heads + head, gates_bf16)), b = gate(beta, int64_t(row) * heads + head, gates_bf16);
        const uint2 raw = *reinterpret_cast<const uint2*>(v + (int64_t(row) * heads + head) * dv + column);
        float kv[ROWS], kq = 0.f;
        float4 sk = make_float4(0.f, 0.f, 0.f, 0.f), sq = sk;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            kv[i] = bf2f(kr[group + i * STEP_GROUPS]);
            const float qv = bf2f(qr[group + i * STEP_GROUPS]);
            kq += kv[i] * qv;
            sk.x += s[i].x * kv[i], sk.y += s[i].y * kv[i], sk.z += s[i].z * kv[i], sk.w += s[i].w * kv[i];
            sq.x += s[i].x * qv, sq.y += s[i].y * qv, sq.z += s[i].z * qv, sq.w += s[i].w * qv;
        }
#pragma unroll
        for (int m = 8; m < 32; m <<= 1) {
            sk.x += __shfl_xor_sync(FULL, sk.x, m), sk.y += __shfl_xor_sync(FULL, sk.y, m);
            sk.z += __shfl_xor_sync(FULL, sk.z, m), sk.w += __shfl_xor_sync(FULL, sk.w, m);
            sq.x += __shfl_xor_sync(FULL, sq.x, m), sq.y += __shfl_xor_sync(FULL, sq.y, m);
            sq.z += __shfl_xor_sync(FULL, sq.z, m), sq.w += __shfl_xor_sync(FULL, sq.w, m);
            kq += __shfl_xor_sync(FULL, kq, m);
        }
        if (lane < 8) part[warp][0][lane] = sk, part[warp][1][lane] = sq;
        if (lane == 0) part_kq[warp] = kq;
        int next = 0x7fffffff;
        if (slots)
            for (int i = row + 1 + thread; i < batch; i += STEP_THREADS)
                if (__ldg(slots + i) == slot) {
                    next = i;
                    break;
                }
        next = __reduce_min_sync(FULL, next);
        if (lane == 0) next_of[warp] = next;
        __syncthreads();
        sk = part[0][0][lane & 7], sq = part[0][1][lane & 7], kq = part_kq[0], next = next_of[0];
#pragma unroll
        for (int w = 1; w < STEP_THREADS / 32; ++w) {
            const float4 x = part[w][0][lane & 7], y = part[w][1][lane & 7];
            sk.x += x.x, sk.y += x.y, sk.z += x.z, sk.w += x.w;
            sq.x += y.x, sq.y += y.y, sq.z += y.z, sq.w += y.w;
            kq += part_kq[w];
            next = min(next, next_of[w]);
        }
        const float4 u = make_float4(b * (low_half(raw.x) - decay * sk.x), b * (high_half(raw.x) - decay * sk.y),
                                     b * (low_half(raw.y) - decay * sk.z), b * (high_half(raw.y) - decay * sk.w));
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            s[i] = make_float4(decay * s[i].x + kv[i] * u.x, decay * s[i].y + kv[i] * u.y, decay * s[i].z + kv[i] * u.z, decay * s[i].w + kv[i] * u.w);
        if (thread < 8)
            *reinterpret_cast<uint2*>(out + (int64_t(row) * heads + head) * dv + column) =
                make_uint2(pack2(scale * (decay * sq.x + kq * u.x), scale * (decay * sq.y + kq * u.y)),
                           pack2(scale * (decay * sq.z + kq * u.z), scale * (decay * sq.w + kq * u.w)));
        if (next >= batch) break;
        row = next;
        __syncthreads();  // the sums are free for the next token
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) at[i * stride] = s[i];
}
}  // namespace

cudaError_t launch_delta_step(const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v, const void* g, const void* beta,
                              bool gates_bf16, float scale, float* state, const int* slots, int64_t pool, int batch, int key_heads,
                              int heads, int d, int dv, __nv_bfloat16* out, cudaStream_t stream) {
    const dim3 grid(dv / STEP_COLUMNS, heads, batch);
    auto* kernel = d == 32 ? delta_step_kernel<32> : d == 64 ? delta_step_kernel<64> : delta_step_kernel<128>;
    KernelTimer timer("delta_step", stream);
    kernel<<<grid, STEP_THREADS, 0, stream>>>(q, k, v, g, beta, gates_bf16, scale, state, slots, pool, batch, key_heads, heads, dv, out);
    return cudaGetLastError();
}

}  // namespace dism
