// Gradients of one chunk of the gated delta rule on tcgen05 (D and DV of 64 or 128; delta_backward.cu has the other widths and the
// formulas).  One CTA per chunk and key head walks the value heads that share the key head.
//
// Every product has M = 128: operands that meet the same right side are stacked.
//     Z  = [dO; dY] X^T        QK = [Q; K] K^T        (128 x 64)
//     U1 = [dO; dY] S0^T       U2 = [dP~; dL~] K      (128 x D)
//     V1 = X dS1^T             V2 = dL~^T K + dP~^T Q  (64 x D; the rows stand twice, the left operand's other half being itself)
// Rows 0-63 of Z, QK, U are the queries' part, rows 64-127 the keys', so a thread, which owns a row of tensor memory, forms
//     dQ = scale e^G U1 + U2        or        dK = -e^G U1 + U2 + e^{G_63 - G} b V1 + V2
// and all row sums of dG without a shuffle; column sums take one transposing reduction over the warp.  Each tile lies in shared
// memory once and is read K-major or MN-major as a product needs it; [dP~; dL~] goes back there as bf16.
//
// 192 KB in and 32 KB out of memory per chunk and head at D = DV = 128 against about 1200 clocks of tensor cores: the loads bound it.
#include "delta_common.cuh"
#include "tensor_memory.cuh"

namespace dism {
namespace {

__device__ int delta_gradient_fault;

constexpr int GRADIENT_THREADS = 256;
constexpr uint32_t TM_Z = 0, TM_QK = 64, TM_U2 = 0, TM_U1 = 128, TM_V1 = 256, TM_V2 = 384, TM_COLUMNS = 512;  // U2 follows Z and QK

template <int D, int DV>
struct GradientTiles {
    static constexpr int STACK = 128 * 128;  // bytes of 128 rows by 64 columns
    static constexpr int QK = 0, GRAD = QK + D / 64 * STACK, PAIRS = GRAD + DV / 64 * STACK, X = PAIRS + STACK, S0 = X + DV * 128, DS = S0 + 2 * D * DV;
    static constexpr int ROWS = DS + 2 * D * DV, SUMS = ROWS + ROW_VALUES * 4;
    // floats: rows of M [2][128], its columns [4][64], columns of b [2][64], state terms of dG [2][128], of dG_63 [2][64], <dS1, S0> [8]
    static constexpr int ROW_SUM = 0, COLUMN_SUM = 256, BETA_SUM = COLUMN_SUM + 256, STATE_SUM = BETA_SUM + 128, LAST_SUM = STATE_SUM + 256, DOT = LAST_SUM + 128;
    static constexpr int BYTES = SUMS + (DOT + 8) * 4 + 1024;  // and room to start at a multiple of 1024
};
struct GradientControl {
    uint64_t first, second;
    uint32_t tensor_memory;
    int abort;
};

// `count` of 64 strided rows of WIDTH elements into swizzled blocks of 64 columns, STACK bytes apart; zeros behind them
template <int WIDTH, int STACK>
__device__ __forceinline__ void load_stack(unsigned tile, const char* global, int64_t stride, int count, int thread) {
    constexpr int PIECES = WIDTH / 8, STEP = GRADIENT_THREADS / PIECES;
    const int first = thread / PIECES, piece = thread % PIECES;
    const unsigned to = tile + (piece >> 3) * STACK + first * 128;
    const char* from = global + first * stride + piece * 16;
#pragma unroll
    for (int row = 0; row < CHUNK; row += STEP) {
        const bool inside = first + row < count;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + row * 128 + (((piece & 7) ^ ((first + row) & 7)) * 16)),
                     "l"(inside ? from : global), "r"(inside ? 16 : 0) : "memory");
        from += STEP * stride;
    }
}
// ROWS x WIDTH elements kept as 8 x 8 blocks into swizzled blocks of 64 columns
template <int ROWS, int WIDTH>
__device__ __forceinline__ void load_blocked(unsigned tile, const __nv_bfloat16* global, int thread) {
#pragma unroll
    for (int i = thread; i < ROWS * WIDTH / 8; i += GRADIENT_THREADS) {
        const int block = i >> 3, r = i & 7, column = block % (WIDTH / 8), row = block / (WIDTH / 8) * 8 + r;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tile + (column >> 3) * (ROWS * 128) + row * 128 + (((column & 7) ^ r) * 16)),
                     "l"(global + i * 8) : "memory");
    }
}
// v[i] of every lane is summed over the warp for each i; lane l keeps the sum of i = l
__device__ __forceinline__ float transposing_sum(float (&v)[32], int lane) {
#pragma unroll
    for (int step = 16; step; step >>= 1) {
        const bool upper = lane & step;
#pragma unroll
        for (int i = 0; i < step; ++i) {
            const float kept = upper ? v[i + step] : v[i], sent = upper ? v[i] : v[i + step];
            v[i] = kept + __shfl_xor_sync(FULL, sent, step);
        }
    }
    return v[0];
}

template <int D, int DV>
__global__ void __launch_bounds__(GRADIENT_THREADS, 1) delta_gradient_tensor_kernel(DeltaShape shape, const __nv_bfloat16* __restrict__ q,
                                                                                    const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ dout,
                                                                                    const __nv_bfloat16* __restrict__ dy, DeltaSaved saved,
                                                                                    const __nv_bfloat16* __restrict__ dstates, const float* __restrict__ dbeta_parts,
                                                                                    __nv_bfloat16* __restrict__ dq, __nv_bfloat16* __restrict__ dk,
                                                                                    void* __restrict__ dg, void* __restrict__ dbeta) {
    using Tiles = GradientTiles<D, DV>;
    constexpr int STACK = Tiles::STACK, HALF = STACK / 2, COLUMNS = D / 2;
    extern __shared__ unsigned char shared_raw[];
    unsigned char* shared = shared_raw + ((1024 - (tm_address(shared_raw) & 1023)) & 1023);
    __shared__ GradientControl control;
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31, key_head = blockIdx.y, group = shape.heads / shape.key_heads;
    int64_t row;
    int count;
    const int64_t slot = blockIdx.x;
    shape.layout.chunk(slot, row, count);
    if (count == 0) return;
    const uint32_t base = tm_address(shared);
    const float* rows = reinterpret_cast<const float*>(shared + Tiles::ROWS);
    float* sums = reinterpret_cast<float*>(shared + Tiles::SUMS);
    const int64_t key_stride = int64_t(shape.key_heads) * D * 2, value_stride = int64_t(shape.heads) * DV * 2;
    const int64_t key = (row * shape.key_heads + key_head) * D * 2;
    load_stack<D, STACK>(base + Tiles::QK, reinterpret_cast<const char*>(q) + key, key_stride, count, thread);
    load_stack<D, STACK>(base + Tiles::QK + HALF, reinterpret_cast<const char*>(k) + key, key_stride, count, thread);
    if (thread == 0) {
        tm_barrier_init(&control.first, 1), tm_barrier_init(&control.second, 1);
        control.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tm_allocate(&control.tensor_memory, TM_COLUMNS);
    volatile int* abort = &control.abort;
    uint32_t tensor = 0;

    // this thread's row of tensor memory: position t, a query's (part 0) or a key's (part 1); its half of the columns
    const int r = thread & 127, t = r & 63, part = r >> 6, half = warp >> 2;
    float acc[COLUMNS];  // half a row of dQ or dK
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i) acc[i] = 0.f;

    for (int turn = 0; turn < group; ++turn) {
        const int head = key_head * group + turn;
        const int64_t place = slot * shape.heads + head;
        const int64_t value = (row * shape.heads + head) * DV * 2;
        load_stack<DV, STACK>(base + Tiles::GRAD, reinterpret_cast<const char*>(dout) + value, value_stride, count, thread);
        load_stack<DV, STACK>(base + Tiles::GRAD + HALF, reinterpret_cast<const char*>(dy) + value, value_stride, count, thread);
        load_blocked<DV, CHUNK>(base + Tiles::X, saved.x + place * CHUNK * DV, thread);
        load_block<ROW_VALUES * 4, GRADIENT_THREADS>(base + Tiles::ROWS, reinterpret_cast<const char*>(saved.rows + place * ROW_VALUES), thread);
        cp_async_commit();
        load_blocked<DV, D>(base + Tiles::S0, saved.states + place * D * DV, thread);
        load_blocked<DV, D>(base + Tiles::DS, dstates + place * D * DV, thread);
        cp_async_commit();
        cp_async_wait<1>();
        tm_fence_proxy();
        tm_fence_before();
        __syncthreads();
        tm_fence_after();
        tensor = control.tensor_memory;
        const uint32_t lanes = tensor + (uint32_t((warp & 3) * 32) << 16);
        const uint64_t grads = tm_descriptor(base + Tiles::GRAD), keys_across = tm_descriptor(base + Tiles::QK + HALF, STACK);
        if (warp == 0 && !*abort) {
            if (elect_one()) {
                const uint64_t x = tm_descriptor(base + Tiles::X), qk = tm_descriptor(base + Tiles::QK), keys = tm_descriptor(base + Tiles::QK + HALF);
#pragma unroll
                for (int kb = 0; kb < DV / 16; ++kb)
                    tm_mma_shared(tensor + TM_Z, grads + ((kb >> 2) * STACK + (kb & 3) * 32) / 16, x + kb * 2048 / 16, tm_instruction(CHUNK, false, true), kb > 0);
#pragma unroll
                for (int kb = 0; kb < D / 16; ++kb)
                    tm_mma_shared(tensor + TM_QK, qk + ((kb >> 2) * STACK + (kb & 3) * 32) / 16, keys + ((kb >> 2) * STACK + (kb & 3) * 32) / 16,
                                  tm_instruction(CHUNK, false, false), kb > 0);
                tm_commit(&control.first);
            }
            __syncwarp();
        }
        cp_async_wait<0>();
        tm_fence_proxy();
        __syncthreads();
        if (warp == 0 && !*abort) {
            if (elect_one()) {
                const uint64_t s0 = tm_descriptor(base + Tiles::S0, DV * 128), ds = tm_descriptor(base + Tiles::DS, DV * 128), x = tm_descriptor(base + Tiles::X, 0);
#pragma unroll
                for (int kb = 0; kb < DV / 16; ++kb)
                    tm_mma_shared(tensor + TM_U1, grads + ((kb >> 2) * STACK + (kb & 3) * 32) / 16, s0 + kb * 2048 / 16, tm_instruction(D, false, true), kb > 0);
#pragma unroll
                for (int kb = 0; kb < DV / 16; ++kb)
                    tm_mma_shared(tensor + TM_V1, x + kb * 2048 / 16, ds + kb * 2048 / 16, tm_instruction(D, true, true), kb > 0);
            }
            __syncwarp();
        }
        {
            float dot = 0.f;  // <dS1, S0>
            const uint4 *s0 = reinterpret_cast<const uint4*>(shared + Tiles::S0), *ds = reinterpret_cast<const uint4*>(shared + Tiles::DS);
#pragma unroll 4
            for (int i = thread; i < D * DV / 8; i += GRADIENT_THREADS) {
                const uint4 x = s0[i], y = ds[i];
                dot += low_half(x.x) * low_half(y.x) + high_half(x.x) * high_half(y.x) + low_half(x.y) * low_half(y.y) + high_half(x.y) * high_half(y.y);
                dot += low_half(x.z) * low_half(y.z) + high_half(x.z) * high_half(y.z) + low_half(x.w) * low_half(y.w) + high_half(x.w) * high_half(y.w);
            }
#pragma unroll
            for (int m = 16; m; m >>= 1) dot += __shfl_xor_sync(FULL, dot, m);
            if (lane == 0) sums[Tiles::DOT + warp] = dot;
        }
        // dP~ or dL~ of this row: columns 32 half .. 32 half + 31
        tm_wait(&control.first, turn & 1, abort, &delta_gradient_fault, 1);
        tm_fence_after();
        {
            const float high = rows[ROW_HIGH + t], low = rows[ROW_LOW + t];
            float m[32], w[32], row_sum = 0.f;
#pragma unroll
            for (int j = 0; j < 32; j += 16) {
                float z[16], y[16];
                tm_load16(z, lanes + TM_Z + 32 * half + j);
                tm_load16(y, lanes + TM_QK + 32 * half + j);
                tm_wait_load();
                float d[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int s = 32 * half + j + i;
                    const float between = ex2((high - rows[ROW_HIGH + s]) + (low - rows[ROW_LOW + s]));
                    const bool counts = s + part <= t;  // s <= t for queries, s < t for keys
                    const float x = counts ? (part ? -between : shape.scale * between) * z[i] : 0.f;
                    d[i] = x * rows[ROW_BETA + s];
                    w[j + i] = x * y[i];
                    m[j + i] = d[i] * y[i];
                    row_sum += m[j + i];
                }
#pragma unroll
                for (int i = 0; i < 16; i += 8)
                    *reinterpret_cast<uint4*>(shared + Tiles::PAIRS + r * 128 + (((4 * half + (j + i) / 8) ^ (r & 7)) * 16)) =
                        make_uint4(pack2(d[i], d[i + 1]), pack2(d[i + 2], d[i + 3]), pack2(d[i + 4], d[i + 5]), pack2(d[i + 6], d[i + 7]));
            }
            sums[Tiles::ROW_SUM + half * 128 + r] = row_sum;
            sums[Tiles::COLUMN_SUM + (warp & 3) * CHUNK + 32 * half + lane] = transposing_sum(m, lane);
            if (part) sums[Tiles::BETA_SUM + (warp & 1) * CHUNK + 32 * half + lane] = transposing_sum(w, lane);
        }
        tm_fence_proxy();
        tm_fence_before();
        __syncthreads();
        tm_fence_after();
        if (warp == 0 && !*abort) {
            if (elect_one()) {
                const uint64_t pairs = tm_descriptor(base + Tiles::PAIRS), p_across = tm_descriptor(base + Tiles::PAIRS, 0), l_across = tm_descriptor(base + Tiles::PAIRS + HALF, 0);
                const uint64_t queries_across = tm_descriptor(base + Tiles::QK, STACK);
#pragma unroll
                for (int kb = 0; kb < CHUNK / 16; ++kb)
                    tm_mma_shared(tensor + TM_U2, pairs + kb * 32 / 16, keys_across + kb * 2048 / 16, tm_instruction(D, false, true), kb > 0);
#pragma unroll
                for (int kb = 0; kb < CHUNK / 16; ++kb)
                    tm_mma_shared(tensor + TM_V2, l_across + kb * 2048 / 16, keys_across + kb * 2048 / 16, tm_instruction(D, true, true), kb > 0);
#pragma unroll
                for (int kb = 0; kb < CHUNK / 16; ++kb)
                    tm_mma_shared(tensor + TM_V2, p_across + kb * 2048 / 16, queries_across + kb * 2048 / 16, tm_instruction(D, true, true), true);
                tm_commit(&control.second);
            }
            __syncwarp();
        }
        tm_wait(&control.second, turn & 1, abort, &delta_gradient_fault, 2);
        tm_fence_after();
        {
            const float decay = rows[ROW_DECAY + t], f1 = part ? -decay : shape.scale * decay, f2 = rows[ROW_WRITE + t];
            float state_sum = 0.f, last_sum = 0.f;
            const unsigned char* own = shared + Tiles::QK + (half * COLUMNS >> 6) * STACK + r * 128;  // the row of Q or K
#pragma unroll
            for (int j = 0; j < COLUMNS; j += 16) {
                const int column = half * COLUMNS + j;
                float u1[16], u2[16], v1[16], v2[16];
                tm_load16(u1, lanes + TM_U1 + column);
                tm_load16(u2, lanes + TM_U2 + column);
                if (part) {
                    tm_load16(v1, lanes + TM_V1 + column);
                    tm_load16(v2, lanes + TM_V2 + column);
                }
                const int piece = (column & 63) / 8;
                const uint4 x0 = *reinterpret_cast<const uint4*>(own + ((piece ^ (r & 7)) * 16)), x1 = *reinterpret_cast<const uint4*>(own + (((piece + 1) ^ (r & 7)) * 16));
                const uint32_t x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
                tm_wait_load();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float own_value = i & 1 ? high_half(x[i / 2]) : low_half(x[i / 2]);
                    const float a = f1 * u1[i];
                    state_sum += a * own_value;
                    acc[j + i] += a + u2[i];
                    if (part) {
                        const float b = f2 * v1[i];
                        last_sum += b * own_value;
                        acc[j + i] += b + v2[i];
                    }
                }
            }
            sums[Tiles::STATE_SUM + half * 128 + r] = state_sum;
            if (part) sums[Tiles::LAST_SUM + half * CHUNK + t] = last_sum;
        }
        tm_fence_before();
        __syncthreads();
        if (warp == 0) {
            float here[2], last = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int p = 2 * lane + e;
                const float tail = sums[Tiles::LAST_SUM + p] + sums[Tiles::LAST_SUM + CHUNK + p];
                float x = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x += (sums[Tiles::ROW_SUM + i * CHUNK + p] - sums[Tiles::COLUMN_SUM + i * CHUNK + p]) + sums[Tiles::STATE_SUM + i * CHUNK + p];
                here[e] = x - tail;
                last += tail;
                float b = sums[Tiles::BETA_SUM + p] + sums[Tiles::BETA_SUM + CHUNK + p];
                const int64_t stride = shape.layout.slots() * shape.heads * CHUNK;
#pragma unroll
                for (int i = 0; i < DV / 16; ++i) b += __ldg(dbeta_parts + i * stride + place * CHUNK + p);
                if (p < count) {
                    const int64_t index = (row + p) * shape.heads + head;
                    if (shape.gates_bf16) static_cast<__nv_bfloat16*>(dbeta)[index] = __float2bfloat16(b);
                    else static_cast<float*>(dbeta)[index] = b;
                }
            }
#pragma unroll
            for (int m = 16; m; m >>= 1) last += __shfl_xor_sync(FULL, last, m);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) dot += sums[Tiles::DOT + i];
            last += rows[ROW_DECAY + CHUNK - 1] * dot;
            if (lane == 31) here[1] += last;
            here[0] += here[1];
            float after = here[0];
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const float other = __shfl_down_sync(FULL, after, s);
                if (lane + s < 32) after += other;
            }
            after -= here[0];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int p = 2 * lane + e;
                if (p < count) {
                    const int64_t index = (row + p) * shape.heads + head;
                    // a decay that is zero in 32 bits has no gradient; the sum would leave the roundings of terms that cancel
                    const float *high = rows + ROW_HIGH, *low = rows + ROW_LOW;
                    const float step = p ? (high[p] - high[p - 1]) + (low[p] - low[p - 1]) : high[0];
                    const float x = step < -149.f ? 0.f : after + here[e];
                    if (shape.gates_bf16) static_cast<__nv_bfloat16*>(dg)[index] = __float2bfloat16(x);
                    else static_cast<float*>(dg)[index] = x;
                }
            }
        }
        if (turn + 1 < group) __syncthreads();  // tiles and sums are free for the next head
    }
    if (t < count) {
        __nv_bfloat16* to = (part ? dk : dq) + ((row + t) * shape.key_heads + key_head) * D + half * COLUMNS;
#pragma unroll
        for (int i = 0; i < COLUMNS; i += 8)
            *reinterpret_cast<uint4*>(to + i) = make_uint4(pack2(acc[i], acc[i + 1]), pack2(acc[i + 2], acc[i + 3]), pack2(acc[i + 4], acc[i + 5]), pack2(acc[i + 6], acc[i + 7]));
    }
    __syncthreads();
    if (control.abort) __nanosleep(1000000);  // products in flight end before their memory is given back
    if (warp == 0) {
        tm_fence_after();
        tm_free(tensor, TM_COLUMNS);
    }
}

template <int D, int DV>
cudaError_t launch(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    constexpr int BYTES = GradientTiles<D, DV>::BYTES;
    auto* kernel = delta_gradient_tensor_kernel<D, DV>;
    if (cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES)) return status;
    KernelTimer timer("delta_gradient", stream);
    kernel<<<dim3(unsigned(shape.layout.slots()), shape.key_heads), GRADIENT_THREADS, BYTES, stream>>>(
        shape, x.q, x.k, x.dout, x.dv, saved, x.dstates, x.dbeta_parts, x.dq, x.dk, x.dg, x.dbeta);
    return cudaGetLastError();
}
}  // namespace

cudaError_t launch_delta_gradient_tensor(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    if (shape.d == 64) return shape.dv == 64 ? launch<64, 64>(shape, x, saved, stream) : launch<64, 128>(shape, x, saved, stream);
    return shape.dv == 64 ? launch<128, 64>(shape, x, saved, stream) : launch<128, 128>(shape, x, saved, stream);
}

cudaError_t read_delta_fault(int* code) {
    if (cudaError_t status = cudaMemcpyFromSymbol(code, delta_gradient_fault, sizeof(int))) return status;
    const int zero = 0;
    return cudaMemcpyToSymbol(delta_gradient_fault, &zero, sizeof(int));
}

}  // namespace dism
