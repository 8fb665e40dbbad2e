// Gradients of the chunks of the gated delta rule on tcgen05 (D and DV of 64 or 128; delta_backward.cu has the other widths and the
// formulas).  One CTA per SM walks (chunk, key head) units and, in each, the value heads that share the key head.
//
// Every product has M = 128: operands that meet the same right side are stacked.
//     Z  = [dO; dY] X^T        QK = [Q; K] K^T        (128 x 64)
//     U1 = [dO; dY] S0^T       U2 = [dP~; dL~] K      (128 x D)
//     V1 = X dS1^T             V2 = dL~^T K + dP~^T Q  (64 x D, in rows 64-127; what stands in the rows above is not read)
// Rows 0-63 of Z, QK, U are the queries' part, rows 64-127 the keys', so a thread, which owns a row of tensor memory, forms
//     dQ = scale e^G U1 + U2        or        dK = -e^G U1 + U2 + e^{G_63 - G} b V1 + V2
// and all row sums of dG without a shuffle; column sums take one transposing reduction over the warp.  <dS1, S0> is the trace of one
// more product.  Each tile lies in shared memory once and is read K-major or MN-major as a product needs it: Q, K, dO, dY and the
// pairs [dP~; dL~] swizzled, X and the states in the 8 x 8 blocks in which they were kept, so that they arrive as three bulk copies.
//
// What bounds it: 148 KB in and 32 KB out of memory per chunk and head at D = DV = 128, against about 2300 clocks of tensor cores (both
// operands come from shared memory: 6 to 8 KB an instruction).  Eight warps work on the rows; one issues products, one loads
// (boxes of tensor maps; where a chunk ends inside a tile the rows behind it, another document's, are made zeros), one puts the 64 values each of dg and db together.  The
// end of Z, QK, U1, V1 and the trace frees every tile but Q, K (of which there are two) and the pairs, and the next item's loads run
// behind the rest of this one.
// 203 us for 5120 items of D = DV = 128 (16 x 2048 positions, 10 heads): 180 KB in and out an item, its intermediates
// included, 4.6 TB/s or 0.72 of the measured copy rate; 113 us for 2 x 8192, 16 heads of 64.  With a tensor pipe at 22 % and DRAM at 39 % (a
// quarter of that size) it is bound by the latency of an item's phases.  Steps on the way, same shape: mma.sync tiles 511 us, one CTA an item on tcgen05 433, the next item's loads
// behind the present one 281, loops rolled for the instruction cache 262, whole-line stores 249, boxes and roles 212.
#include "delta_common.cuh"
#include "tensor_memory.cuh"

namespace dism {
namespace {

__device__ int delta_gradient_fault;

constexpr int WORK_WARPS = 8, LOAD_WARP = 8, MMA_WARP = 9, GATE_WARP = 10, GRADIENT_THREADS = 384;
// columns of tensor memory: U2 follows Z and QK, V2 the product whose trace is <dS1, S0>
constexpr uint32_t TM_Z = 0, TM_QK = 64, TM_U2 = 0, TM_U1 = 128, TM_V1 = 256, TM_V2 = 384, TM_TRACE = 384, TM_COLUMNS = 512;

template <int D, int DV>
struct GradientTiles {
    static constexpr int STACK = 128 * 128;  // bytes of 128 rows by 64 columns
    static constexpr int STATE = 2 * D * DV;
    // the room of the pairs is also that of dQ and dK on their way out: 32 rows by half of D for each of the eight warps
    static constexpr int QK = 0, GRAD = QK + 2 * (D / 64) * STACK, PAIRS = GRAD + DV / 64 * STACK, X = PAIRS + D / 64 * STACK, S0 = X + DV * 128, DS = S0 + STATE;
    static constexpr int ROWS = DS + STATE, SUMS = ROWS + 2 * ROW_VALUES * 4;  // two of each, an item apart
    // floats: rows of M [2][128], columns of M / b [4][64], state terms of dG [2][128], of dG_63 [2][64], <dS1, S0> [4]
    static constexpr int ROW_SUM = 0, COLUMN_SUM = 256, STATE_SUM = COLUMN_SUM + 256, LAST_SUM = STATE_SUM + 256, DOT = LAST_SUM + 128, SUM_VALUES = DOT + 4;
    static constexpr int BYTES = SUMS + 2 * SUM_VALUES * 4 + 1024;  // and room to start at a multiple of 1024
};
struct GradientControl {
    // Loads; the two groups of products; operands and sums of the rows; dg and db.  Where a waiter could be a whole item late (it is held up
    // by nothing the next item waits for), items take turns on two barriers, so that no phase can pass unseen.
    uint64_t loaded[2], tail, first, second, pairs, done[2], gated[2];
    uint32_t tensor_memory;
    int abort;
};

// One warp: zeros in rows `count` .. 63 of BLOCKS swizzled blocks of 64 columns, `apart` bytes from one another
template <int BLOCKS>
__device__ __forceinline__ void clear_tail(unsigned char* tile, int apart, int count, int lane) {
    for (int i = count * 8 + lane; i < CHUNK * 8; i += 32)
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) *reinterpret_cast<uint4*>(tile + j * apart + i * 16) = make_uint4(0, 0, 0, 0);
}
// The items of a CTA in order: of every gridDim.x-th (slot, key head) with positions, the value heads.
struct Items {
    int slot, key_head, turn;
    int64_t row;
    int count, slots, step_slots, step_heads;
    __device__ Items(const DeltaShape& shape)
        : slot(blockIdx.x / shape.key_heads), key_head(blockIdx.x % shape.key_heads), turn(0), slots(int(shape.layout.slots())),
          step_slots(gridDim.x / shape.key_heads), step_heads(gridDim.x % shape.key_heads) {
        settle(shape);
    }
    __device__ void settle(const DeltaShape& shape) {
        for (; slot < slots; advance(shape)) {
            shape.layout.chunk(slot, row, count);
            if (count > 0) break;
        }
    }
    __device__ void advance(const DeltaShape& shape) {
        slot += step_slots, key_head += step_heads;
        if (key_head >= shape.key_heads) key_head -= shape.key_heads, ++slot;
    }
    __device__ bool valid() const { return slot < slots; }
    __device__ bool last_head(const DeltaShape& shape) const { return (turn + 1) * shape.key_heads >= shape.heads; }
    __device__ int head(const DeltaShape& shape) const { return key_head * (shape.heads / shape.key_heads) + turn; }
    __device__ void next(const DeltaShape& shape) {
        if (!last_head(shape)) {
            ++turn;
            return;
        }
        turn = 0;
        advance(shape);
        settle(shape);
    }
};
__device__ __forceinline__ void factors(float (&f)[16], const float* from) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(f + 4 * i) = reinterpret_cast<const float4*>(from)[i];
}
// v[i] of every lane is summed over the warp for each i; lane l is left with the sum of i = l / 2
__device__ __forceinline__ float transposing_sum(float (&v)[16], int lane) {
#pragma unroll
    for (int step = 8; step; step >>= 1) {
        const bool upper = lane & (2 * step);
#pragma unroll
        for (int i = 0; i < step; ++i) {
            const float kept = upper ? v[i + step] : v[i], sent = upper ? v[i] : v[i + step];
            v[i] = kept + __shfl_xor_sync(FULL, sent, 2 * step);
        }
    }
    return v[0] + __shfl_xor_sync(FULL, v[0], 1);
}

// SHARED: several value heads read a key head, whose gradients are summed in registers.  The loops over columns are rolled where
// registers allow it: the loop over the items has to stay in the instruction cache (unrolled, at 62 KB, it ran at 17 000 clocks an item).
template <int D, int DV, bool SHARED>
__global__ void __launch_bounds__(GRADIENT_THREADS, 1) delta_gradient_tensor_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                                                                                    const __grid_constant__ CUtensorMap dout_map, const __grid_constant__ CUtensorMap dy_map,
                                                                                    DeltaShape shape, DeltaSaved saved,
                                                                                    const __nv_bfloat16* __restrict__ dstates, const float* __restrict__ dbeta_parts,
                                                                                    __nv_bfloat16* __restrict__ dq, __nv_bfloat16* __restrict__ dk,
                                                                                    void* __restrict__ dg, void* __restrict__ dbeta) {
    using Tiles = GradientTiles<D, DV>;
    constexpr int STACK = Tiles::STACK, HALF = STACK / 2, COLUMNS = D / 2;
    extern __shared__ unsigned char shared_raw[];
    unsigned char* shared = shared_raw + ((1024 - (tm_address(shared_raw) & 1023)) & 1023);
    __shared__ GradientControl control;
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    if (shape.layout.cu) clear_gradients<GRADIENT_THREADS>(shape, dq, dk, dg, dbeta, blockIdx.x, gridDim.x, thread);
    Items items(shape);
    if (!items.valid()) return;
    const uint32_t base = tm_address(shared);
    if (thread == 0) {
        for (int i = 0; i < 2; ++i) tm_barrier_init(&control.loaded[i], 1), tm_barrier_init(&control.done[i], WORK_WARPS), tm_barrier_init(&control.gated[i], 1);
        tm_barrier_init(&control.tail, 1), tm_barrier_init(&control.first, 1), tm_barrier_init(&control.second, 1);
        tm_barrier_init(&control.pairs, WORK_WARPS);
        control.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tm_allocate(&control.tensor_memory, TM_COLUMNS);
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    volatile int* abort = &control.abort;
    const uint32_t tensor = control.tensor_memory;
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return tm_wait(bar, parity, abort, &delta_gradient_fault, code, shape.wait_tries); };
    auto rows_of = [&](int item) { return reinterpret_cast<const float*>(shared + Tiles::ROWS + (item & 1) * ROW_VALUES * 4); };
    auto sums_of = [&](int item) { return reinterpret_cast<float*>(shared + Tiles::SUMS) + (item & 1) * Tiles::SUM_VALUES; };
    // 168 registers a thread at launch: the rows take 208, issue and loads 80
    if (warp >= WORK_WARPS) {
        tm_fewer_registers<80>();
        uint64_t* flight = nullptr;  // the barrier of the role's last copies or products
        uint32_t flight_parity = 0;
        if (warp == MMA_WARP) {
            for (int item = 0, keys = 0; items.valid(); ++item) {
                const uint32_t qk_tile = base + Tiles::QK + keys * (D / 64 * STACK);
                const uint64_t keys_across = tm_descriptor(qk_tile + HALF, STACK);
                const bool ok = wait(&control.loaded[item & 1], (item >> 1) & 1, 1) &&
                          (item == 0 || wait(&control.done[(item - 1) & 1], ((item - 1) >> 1) & 1, 3));
                if (!__all_sync(FULL, ok)) break;
                tm_fence_after();
                if (tm_elect()) {
                    const uint64_t grads = tm_descriptor(base + Tiles::GRAD), x = tm_block_descriptor(base + Tiles::X, 128, CHUNK * 16);
                    const uint64_t queries = tm_descriptor(qk_tile), own_keys = tm_descriptor(qk_tile + HALF);
                    const uint64_t s0 = tm_block_descriptor(base + Tiles::S0, 128, D * 16), ds = tm_block_descriptor(base + Tiles::DS, 128, D * 16);
#pragma unroll 2
                    for (int kb = 0; kb < DV / 16; ++kb)
                        tm_mma_shared(tensor + TM_Z, grads + ((kb >> 2) * STACK + (kb & 3) * 32) / 16, x + kb * CHUNK * 2, tm_instruction(CHUNK, false, true), kb > 0);
#pragma unroll 2
                    for (int kb = 0; kb < D / 16; ++kb)
                        tm_mma_shared(tensor + TM_QK, queries + ((kb >> 2) * STACK + (kb & 3) * 32) / 16, own_keys + ((kb >> 2) * STACK + (kb & 3) * 32) / 16,
                                      tm_instruction(CHUNK, false, false), kb > 0);
#pragma unroll 2
                    for (int kb = 0; kb < DV / 16; ++kb)
                        tm_mma_shared(tensor + TM_U1, grads + ((kb >> 2) * STACK + (kb & 3) * 32) / 16, s0 + kb * D * 2, tm_instruction(D, false, true), kb > 0);
                    // X as rows 64-127: eight blocks before it begins
#pragma unroll 2
                    for (int kb = 0; kb < DV / 16; ++kb)
                        tm_mma_shared(tensor + TM_V1, x - 1024 / 16 + kb * CHUNK * 2, ds + kb * D * 2, tm_instruction(D, true, true), kb > 0);
#pragma unroll 2
                    for (int kb = 0; kb < DV / 16; ++kb)
                        tm_mma_shared(tensor + TM_TRACE, s0 + kb * D * 2, ds + kb * D * 2, tm_instruction(D, true, true), kb > 0);
                    tm_commit(&control.first);
                }
                __syncwarp();
                flight = &control.first, flight_parity = item & 1;
                if (!__all_sync(FULL, wait(&control.pairs, item & 1, 4))) break;
                tm_fence_after();
                if (tm_elect()) {
                    const uint64_t pairs = tm_descriptor(base + Tiles::PAIRS), p_across = tm_descriptor(base + Tiles::PAIRS, 0), l_across = tm_descriptor(base + Tiles::PAIRS + HALF, 0);
                    const uint64_t queries_across = tm_descriptor(qk_tile, STACK);
#pragma unroll 2
                    for (int kb = 0; kb < CHUNK / 16; ++kb)
                        tm_mma_shared(tensor + TM_U2, pairs + kb * 32 / 16, keys_across + kb * 2048 / 16, tm_instruction(D, false, true), kb > 0);
#pragma unroll 2
                    for (int kb = 0; kb < CHUNK / 16; ++kb)
                        tm_mma_shared(tensor + TM_V2, l_across + kb * 2048 / 16, keys_across + kb * 2048 / 16, tm_instruction(D, true, true), kb > 0);
#pragma unroll 2
                    for (int kb = 0; kb < CHUNK / 16; ++kb)
                        tm_mma_shared(tensor + TM_V2, p_across + kb * 2048 / 16, queries_across + kb * 2048 / 16, tm_instruction(D, true, true), true);
                    tm_commit(&control.second);
                }
                __syncwarp();
                flight = &control.second;
                if (items.last_head(shape)) keys ^= 1;
                items.next(shape);
            }
        } else if (warp == LOAD_WARP) {
            for (int item = 0, keys = 0, tails = 0; items.valid(); ++item) {
                if (item > 0 && !__all_sync(FULL, wait(&control.first, (item - 1) & 1, 5))) break;                    // the tiles are free
                if (item > 1 && !__all_sync(FULL, wait(&control.gated[item & 1], ((item - 2) >> 1) & 1, 2))) break;  // and the table of two items ago
                const int head = items.head(shape), keys_at = Tiles::QK + keys * (D / 64 * STACK);
                const int64_t place = int64_t(items.slot) * shape.heads + head;
                const bool new_keys = items.turn == 0, partial = items.count < CHUNK;
                uint64_t *loaded = &control.loaded[item & 1], *boxes = partial ? &control.tail : loaded;
                const uint32_t box_bytes = (DV / 64 + (new_keys ? D / 64 : 0)) * STACK, copy_bytes = DV * 128 + 2 * Tiles::STATE + ROW_VALUES * 4;
                if (lane == 0) {
                    const int at = int(items.row);
                    tm_expect(boxes, partial ? box_bytes : box_bytes + copy_bytes);
#pragma unroll
                    for (int j = 0; j < DV / 64; ++j) {
                        tm_load_box(base + Tiles::GRAD + j * STACK, &dout_map, head * DV + j * 64, at, boxes);
                        tm_load_box(base + Tiles::GRAD + j * STACK + HALF, &dy_map, head * DV + j * 64, at, boxes);
                    }
#pragma unroll
                    for (int j = 0; j < D / 64 && new_keys; ++j) {
                        tm_load_box(base + keys_at + j * STACK, &q_map, items.key_head * D + j * 64, at, boxes);
                        tm_load_box(base + keys_at + j * STACK + HALF, &k_map, items.key_head * D + j * 64, at, boxes);
                    }
                }
                __syncwarp();
                flight = boxes, flight_parity = (partial ? tails : item >> 1) & 1;
                if (partial) {  // the rows behind a chunk that ends inside its tile are another document's
                    if (!__all_sync(FULL, wait(&control.tail, tails & 1, 10))) break;
                    ++tails;
                    clear_tail<DV / 64>(shared + Tiles::GRAD, STACK, items.count, lane);
                    clear_tail<DV / 64>(shared + Tiles::GRAD + HALF, STACK, items.count, lane);
                    if (new_keys) {
                        clear_tail<D / 64>(shared + keys_at, STACK, items.count, lane);
                        clear_tail<D / 64>(shared + keys_at + HALF, STACK, items.count, lane);
                    }
                    tm_fence_proxy();  // written through the generic proxy, read by the tensor cores
                    __syncwarp();
                }
                if (lane == 0) {
                    if (partial) tm_expect(loaded, copy_bytes);
                    tm_copy(base + Tiles::X, saved.x + place * CHUNK * DV, DV * 128, loaded);
                    tm_copy(base + Tiles::S0, saved.states + place * D * DV, Tiles::STATE, loaded);
                    tm_copy(base + Tiles::DS, dstates + place * D * DV, Tiles::STATE, loaded);
                    tm_copy(base + Tiles::ROWS + (item & 1) * ROW_VALUES * 4, saved.rows + place * ROW_VALUES, ROW_VALUES * 4, loaded);
                }
                __syncwarp();
                flight = loaded, flight_parity = (item >> 1) & 1;
                if (items.last_head(shape)) keys ^= 1;
                items.next(shape);
            }
        } else if (warp == GATE_WARP) {
            for (int item = 0; items.valid(); ++item) {
                const int head = items.head(shape);
                const int64_t place = int64_t(items.slot) * shape.heads + head;
                const float *rows = rows_of(item), *sums = sums_of(item);
                float parts[2][DV / 16];  // what the reverse chain left of db
                const int64_t stride = shape.layout.slots() * shape.heads * CHUNK;
#pragma unroll
                for (int i = 0; i < DV / 16; ++i) {
                    const float2 x = __ldg(reinterpret_cast<const float2*>(dbeta_parts + i * stride + place * CHUNK) + lane);
                    parts[0][i] = x.x, parts[1][i] = x.y;
                }
                wait(&control.loaded[item & 1], (item >> 1) & 1, 11);
                wait(&control.done[item & 1], (item >> 1) & 1, 6);
                const bool lost = *abort;
                {
                    float here[2], last = 0.f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int p = 2 * lane + e;
                        const float tail = sums[Tiles::LAST_SUM + p] + sums[Tiles::LAST_SUM + CHUNK + p], beta = rows[ROW_BETA + p];
                        float x = 0.f, b = 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            x += (sums[Tiles::ROW_SUM + i * CHUNK + p] - __fmul_rn(beta, sums[Tiles::COLUMN_SUM + i * CHUNK + p])) + sums[Tiles::STATE_SUM + i * CHUNK + p];
                        here[e] = x - tail;
                        last += tail;
#pragma unroll
                        for (int i = 0; i < DV / 16; ++i) b += parts[e][i];
                        b += sums[Tiles::COLUMN_SUM + 2 * CHUNK + p] + sums[Tiles::COLUMN_SUM + 3 * CHUNK + p];
                        if (lost) b = NOT_A_NUMBER;
                        if (p < items.count) {
                            const int64_t index = (items.row + p) * shape.heads + head;
                            if (shape.gates_bf16) static_cast<__nv_bfloat16*>(dbeta)[index] = __float2bfloat16(b);
                            else static_cast<float*>(dbeta)[index] = b;
                        }
                    }
#pragma unroll
                    for (int m = 16; m; m >>= 1) last += __shfl_xor_sync(FULL, last, m);
                    float dot = 0.f;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) dot += sums[Tiles::DOT + i];
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
                        if (p < items.count) {
                            const int64_t index = (items.row + p) * shape.heads + head;
                            // a decay that is zero in 32 bits has no gradient; the sum would leave the roundings of terms that cancel
                            const float *high = rows + ROW_HIGH, *low = rows + ROW_LOW;
                            const float step = p ? (high[p] - high[p - 1]) + (low[p] - low[p - 1]) : high[0];
                            const float x = lost ? NOT_A_NUMBER : step < -149.f ? 0.f : after + here[e];
                            if (shape.gates_bf16) static_cast<__nv_bfloat16*>(dg)[index] = __float2bfloat16(x);
                            else static_cast<float*>(dg)[index] = x;
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) tm_arrive(&control.gated[item & 1]);
                items.next(shape);
            }
        }
        if (flight) tm_settle(flight, flight_parity);
    } else {
        tm_more_registers<208>();
        // this thread's row of tensor memory: position t, a query's (part 0) or a key's (part 1); its half of the columns
        const int r = thread & 127, t = r & 63, part = r >> 6, half = warp >> 2;
        const uint32_t lanes = tensor + (uint32_t((warp & 3) * 32) << 16);
        auto arrive = [&](uint64_t* bar) {
            tm_fence_before();
            __syncwarp();
            if (lane == 0) tm_arrive(bar);
        };
        float acc[SHARED ? COLUMNS : 16];  // half a row of dQ or dK
#pragma unroll
        for (int i = 0; i < COLUMNS && SHARED; ++i) acc[i] = 0.f;
        for (int item = 0, keys = 0; items.valid(); ++item) {
            const float* rows = rows_of(item);
            float* sums = sums_of(item);
            wait(&control.loaded[item & 1], (item >> 1) & 1, 7);
            wait(&control.first, item & 1, 8);
            tm_fence_after();
            // dP~ or dL~ of this row: columns 32 half .. 32 half + 31
            {
                const float high = rows[ROW_HIGH + t], low = rows[ROW_LOW + t];
                const bool lost = *abort;  // then another warp may still have its rows of the last item in the room of the pairs
                float row_sum = 0.f;
#pragma unroll 1
                for (int j = 32 * half; j < 32 * half + 32; j += 16) {
                    float z[16], y[16];
                    tm_load16(z, lanes + TM_Z + j);
                    tm_load16(y, lanes + TM_QK + j);
                    float h[16], l[16], beta[16];
                    factors(h, rows + ROW_HIGH + j);
                    factors(l, rows + ROW_LOW + j);
                    factors(beta, rows + ROW_BETA + j);
                    tm_wait_load();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float between = ex2((high - h[i]) + (low - l[i]));
                        const bool counts = j + i + part <= t;  // s <= t for queries, s < t for keys
                        const float x = counts ? (part ? -between : shape.scale * between) * z[i] : 0.f;
                        z[i] = x * beta[i];
                        y[i] *= x;
                        row_sum += __fmul_rn(beta[i], y[i]);  // as the column sums have it: a pair that cancels in dG is one number
                    }
#pragma unroll
                    for (int i = 0; i < 16 && !lost; i += 8)
                        *reinterpret_cast<uint4*>(shared + Tiles::PAIRS + r * 128 + ((((j + i) / 8) ^ (r & 7)) * 16)) =
                            make_uint4(pack2(z[i], z[i + 1]), pack2(z[i + 2], z[i + 3]), pack2(z[i + 4], z[i + 5]), pack2(z[i + 6], z[i + 7]));
                    const float column = transposing_sum(y, lane);
                    if (!(lane & 1)) sums[Tiles::COLUMN_SUM + (warp & 3) * CHUNK + j + lane / 2] = column;
                }
                sums[Tiles::ROW_SUM + half * 128 + r] = row_sum;
                if (half == 0 && r < D) {  // the trace: element r of this row
                    float dot = 0.f;
#pragma unroll 1
                    for (int j = 0; j < 32; j += 16) {
                        float x[16];
                        tm_load16(x, lanes + TM_TRACE + (warp & 3) * 32 + j);
                        tm_wait_load();
#pragma unroll
                        for (int i = 0; i < 16; ++i) dot += j + i == lane ? x[i] : 0.f;
                    }
#pragma unroll
                    for (int m = 16; m; m >>= 1) dot += __shfl_xor_sync(FULL, dot, m);
                    if (lane == 0) sums[Tiles::DOT + warp] = dot;
                }
            }
            tm_fence_proxy();
            arrive(&control.pairs);
            const bool whole = items.last_head(shape);
            wait(&control.second, item & 1, 9);
            tm_fence_after();
            {
                const float decay = rows[ROW_DECAY + t], f1 = *abort ? NOT_A_NUMBER : part ? -decay : shape.scale * decay, f2 = rows[ROW_WRITE + t];
                float state_sum = 0.f, last_sum = 0.f;
                const unsigned char* own = shared + Tiles::QK + keys * (D / 64 * STACK) + (half * COLUMNS >> 6) * STACK + r * 128;  // the row of Q or K
                constexpr int ROW = 2 * COLUMNS, PIECES = ROW / 16;
                unsigned char* stage = shared + Tiles::PAIRS + warp * 32 * ROW;
                auto take = [&](int j, float* sum) {  // sixteen columns
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
                        sum[i] += a + u2[i];
                        if (part) {
                            const float b = f2 * v1[i];
                            last_sum += b * own_value;
                            sum[i] += b + v2[i];
                        }
                    }
                };
                auto store = [&](int j, const float* sum) {
#pragma unroll
                    for (int i = 0; i < 16; i += 8)
                        *reinterpret_cast<uint4*>(stage + lane * ROW + (((j + i) / 8 ^ piece_key<ROW>(lane)) * 16)) =
                            make_uint4(pack2(sum[i], sum[i + 1]), pack2(sum[i + 2], sum[i + 3]), pack2(sum[i + 4], sum[i + 5]), pack2(sum[i + 6], sum[i + 7]));
                };
                if constexpr (SHARED) {
#pragma unroll
                    for (int j = 0; j < COLUMNS; j += 16) {
                        take(j, acc + j);
                        if (whole) store(j, acc + j);
                    }
                } else {
#pragma unroll 1
                    for (int j = 0; j < COLUMNS; j += 16) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[i] = 0.f;
                        take(j, acc);
                        store(j, acc);
                    }
                }
                sums[Tiles::STATE_SUM + half * 128 + r] = state_sum;
                if (part) sums[Tiles::LAST_SUM + half * CHUNK + t] = last_sum;
                if (whole) {  // whole lines: a thread's own row, piece by piece, would cost the load-store unit a line per lane
                    __syncwarp();
                    const int first = (warp & 1) * 32;
                    __nv_bfloat16* to = (part ? dk : dq) + ((items.row + first) * shape.key_heads + items.key_head) * D + half * COLUMNS;
#pragma unroll 2
                    for (int i = lane; i < 32 * PIECES; i += 32) {
                        const int line = i / PIECES, piece = i % PIECES;
                        const uint4 x = *reinterpret_cast<const uint4*>(stage + line * ROW + ((piece ^ piece_key<ROW>(line)) * 16));
                        if (first + line < items.count) *reinterpret_cast<uint4*>(to + int64_t(line) * shape.key_heads * D + piece * 8) = x;
                    }
                }
            }
            arrive(&control.done[item & 1]);
            if (whole) {
#pragma unroll
                for (int i = 0; i < COLUMNS && SHARED; ++i) acc[i] = 0.f;
                keys ^= 1;
            }
            items.next(shape);
        }
    }
    __syncthreads();
    if (warp == 0) {
        tm_fence_after();
        tm_free(tensor, TM_COLUMNS);
    }
}

template <int D, int DV, bool SHARED>
cudaError_t launch(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    constexpr int BYTES = GradientTiles<D, DV>::BYTES;
    constexpr auto* kernel = delta_gradient_tensor_kernel<D, DV, SHARED>;
    if (cudaError_t status = allow_shared<kernel>(BYTES)) return status;
    const uint64_t rows = shape.layout.cu ? uint64_t(shape.layout.n) : uint64_t(shape.layout.sequences) * shape.layout.n;
    const uint64_t key_width = uint64_t(shape.key_heads) * D, value_width = uint64_t(shape.heads) * DV;
    CUtensorMap q_map, k_map, dout_map, dy_map;
    if (!encode_rows(&q_map, x.q, rows, key_width, key_width, CHUNK) || !encode_rows(&k_map, x.k, rows, key_width, key_width, CHUNK) ||
        !encode_rows(&dout_map, x.dout, rows, value_width, value_width, CHUNK) || !encode_rows(&dy_map, x.dv, rows, value_width, value_width, CHUNK))
        return cudaErrorInvalidValue;
    KernelTimer timer("delta_gradient", stream);
    const int64_t units = shape.layout.slots() * shape.key_heads;
    kernel<<<unsigned(units < device_sm_count() ? units : device_sm_count()), GRADIENT_THREADS, BYTES, stream>>>(
        q_map, k_map, dout_map, dy_map, shape, saved, x.dstates, x.dbeta_parts, x.dq, x.dk, x.dg, x.dbeta);
    return cudaGetLastError();
}
template <int D, int DV>
cudaError_t choose(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    return shape.heads > shape.key_heads ? launch<D, DV, true>(shape, x, saved, stream) : launch<D, DV, false>(shape, x, saved, stream);
}
}  // namespace

cudaError_t launch_delta_gradient_tensor(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    if (shape.d == 64) return shape.dv == 64 ? choose<64, 64>(shape, x, saved, stream) : choose<64, 128>(shape, x, saved, stream);
    return shape.dv == 64 ? choose<128, 64>(shape, x, saved, stream) : choose<128, 128>(shape, x, saved, stream);
}

cudaError_t read_delta_fault(int* code) {
    int chain = 0, reverse = 0;
    const int zero = 0;
    if (cudaError_t status = cudaDeviceSynchronize()) return status;  // the copies alone wait for no non-blocking stream
    if (cudaError_t status = read_chain_fault(&chain)) return status;
    if (cudaError_t status = read_reverse_fault(&reverse)) return status;
    if (cudaError_t status = cudaMemcpyFromSymbol(code, delta_gradient_fault, sizeof(int))) return status;
    if (chain || reverse) *code = chain ? chain : reverse;  // the earlier stage
    return cudaMemcpyToSymbol(delta_gradient_fault, &zero, sizeof(int));
}

}  // namespace dism
