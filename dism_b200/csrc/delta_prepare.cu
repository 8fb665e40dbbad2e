// Chunk matrices of the gated delta rule: T = (I + L diag(b))^-1, P = scale tril(E * Q K^T) and the decay table of every
// chunk of 64 positions and every value head; all independent of one another and of the state.
//
// The inverse of A = I + L diag(b): the four 16 x 16 diagonal tiles by forward substitution in 32 bits (a warp each, a lane a
// column), then twice two neighbouring blocks are joined,
//     [T1 0; T21 T2],   T21 = -T2 A21 T1,
// on the tensor cores.  The joins are computed transposed, Z^T = T1^T A21^T and T21^T = -Z^T T2^T, so that Z stays in registers,
// with every operand as a bf16 pair (three products): the inverse is good to 16 bits, which the exact state needs.  (A substitution of
// all 64 rows, a lane a column, took 132 us where the joined inverse took 80.)
//
// Bound by latency: five CTAs per SM, each a chain of load, products, substitution and two joins with a barrier between (tensor pipe 32 %,
// DRAM 21 %, most stalls at barriers and loads).  78 us for 5120 chunks of D = 128 (16 x 2048 positions, 10 heads): 44 KB in and out
// of memory per chunk, 2.9 TB/s.
#include "delta_common.cuh"

namespace dism {
namespace {

constexpr int PREPARE_THREADS = 128, SQUARE_PITCH = 2 * CHUNK + 16, SQUARE = CHUNK * SQUARE_PITCH, DIAGONAL = 20;

// a*b + a*rest(b) + rest(a)*b for one 16 x 16 by 16 x 8 product of pairs
__device__ __forceinline__ void mma_pairs(float (&c)[4], const unsigned (&a)[4], const unsigned (&a_rest)[4], unsigned b0, unsigned b1, unsigned r0, unsigned r1) {
    mma16816(c, a, b0, b1);
    mma16816(c, a, r0, r1);
    mma16816(c, a_rest, b0, b1);
}

// One 16-column strip (columns `column` .. +15 of T1) of a join of two blocks of SIZE rows at `first` and `first + SIZE`, for the output
// rows `first + SIZE + 16 OUT_FIRST` .. of OUT_TILES tiles.  a and t: matrices in shared memory, the remainders SQUARE bytes behind.
template <int SIZE, int OUT_TILES>
__device__ __forceinline__ void join(unsigned a, unsigned t, int first, int column, int out_first, int lane) {
    constexpr int TILES = SIZE / 16;
    float z[2 * TILES][4];
#pragma unroll
    for (int n = 0; n < 2 * TILES; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[n][e] = 0.f;
    const unsigned t1 = t + (first * SQUARE_PITCH + (first + column) * 2) + cols_first(lane, SQUARE_PITCH);
    const unsigned a21 = a + ((first + SIZE) * SQUARE_PITCH + first * 2) + cols_first(lane, SQUARE_PITCH);
#pragma unroll
    for (int kb = 0; kb < TILES; ++kb) {
        unsigned x[4], x_rest[4];
        ldsm4_trans(x, t1 + kb * 16 * SQUARE_PITCH);
        ldsm4_trans(x_rest, t1 + SQUARE + kb * 16 * SQUARE_PITCH);
#pragma unroll
        for (int np = 0; np < TILES; ++np) {
            unsigned b[4], r[4];
            ldsm4(b, a21 + np * 16 * SQUARE_PITCH + kb * 32);
            ldsm4(r, a21 + SQUARE + np * 16 * SQUARE_PITCH + kb * 32);
            mma_pairs(z[2 * np], x, x_rest, b[0], b[1], r[0], r[1]);
            mma_pairs(z[2 * np + 1], x, x_rest, b[2], b[3], r[2], r[3]);
        }
    }
    float y[2 * OUT_TILES][4];
#pragma unroll
    for (int n = 0; n < 2 * OUT_TILES; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[n][e] = 0.f;
    const unsigned t2 = t + ((first + SIZE + out_first * 16) * SQUARE_PITCH + (first + SIZE) * 2) + cols_first(lane, SQUARE_PITCH);
#pragma unroll
    for (int kb = 0; kb < TILES; ++kb) {
        unsigned x[4], x_rest[4];
        to_operand(x, z[2 * kb], z[2 * kb + 1]);
        to_operand_rest(x_rest, x, z[2 * kb], z[2 * kb + 1]);
#pragma unroll
        for (int np = 0; np < OUT_TILES; ++np) {
            unsigned b[4], r[4];
            ldsm4(b, t2 + np * 16 * SQUARE_PITCH + kb * 32);
            ldsm4(r, t2 + SQUARE + np * 16 * SQUARE_PITCH + kb * 32);
            mma_pairs(y[2 * np], x, x_rest, b[0], b[1], r[0], r[1]);
            mma_pairs(y[2 * np + 1], x, x_rest, b[2], b[3], r[2], r[3]);
        }
    }
    const unsigned to = t + ((first + SIZE + out_first * 16) * SQUARE_PITCH + (first + column) * 2) + cols_first(lane, SQUARE_PITCH);
#pragma unroll
    for (int np = 0; np < OUT_TILES; ++np) {
        float(&y0)[4] = y[2 * np], (&y1)[4] = y[2 * np + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) y0[e] = -y0[e], y1[e] = -y1[e];
        unsigned x[4], x_rest[4];
        to_operand(x, y0, y1);
        to_operand_rest(x_rest, x, y0, y1);
        stsm4_trans(to + np * 16 * SQUARE_PITCH, x[0], x[1], x[2], x[3]);
        stsm4_trans(to + SQUARE + np * 16 * SQUARE_PITCH, x_rest[0], x_rest[1], x_rest[2], x_rest[3]);
    }
}

template <int D>
struct PrepareShared {
    // K and Q; once their products are in registers the same room holds A and T as pairs
    static constexpr int PITCH = 2 * D + 16, TILES = 2 * CHUNK * PITCH > 4 * SQUARE ? 2 * CHUNK * PITCH : 4 * SQUARE;
    static constexpr int TABLE = TILES, DIAGONALS = TABLE + 3 * CHUNK * 4, BYTES = DIAGONALS + 4 * 16 * DIAGONAL * 4;
};

template <int D>
__global__ void __launch_bounds__(PREPARE_THREADS, 5) delta_prepare_kernel(DeltaShape shape, const __nv_bfloat16* __restrict__ q,
                                                                           const __nv_bfloat16* __restrict__ k, const void* __restrict__ g,
                                                                           const void* __restrict__ beta, DeltaSaved saved) {
    using Shared = PrepareShared<D>;
    constexpr int PITCH = Shared::PITCH;
    extern __shared__ __align__(16) unsigned char shared[];
    float* table = reinterpret_cast<float*>(shared + Shared::TABLE);  // G as a pair, then b
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31, head = blockIdx.y;
    const int key_head = head / (shape.heads / shape.key_heads);
    int64_t row;
    int count;
    const int64_t slot = blockIdx.x;
    shape.layout.chunk(slot, row, count);
    if (count == 0) return;
    const unsigned base = smem_address(shared);
    const int64_t stride = int64_t(shape.key_heads) * D * 2, at = (row * shape.key_heads + key_head) * D * 2;
    load_rows<2 * D, PREPARE_THREADS>(base, PITCH, reinterpret_cast<const char*>(k) + at, stride, count, thread);
    load_rows<2 * D, PREPARE_THREADS>(base + CHUNK * PITCH, PITCH, reinterpret_cast<const char*>(q) + at, stride, count, thread);
    cp_async_commit();
    const int64_t place = slot * shape.heads + head;
    if (warp == 0) {
        // G in 64 bits, kept as two floats: its differences stay exact to 32 bits however far the sum has run.  A decay
        // of zero (g of minus infinity) becomes 2^-256, which is zero in 32 bits and leaves the sums finite.
        float* rows = saved.rows + place * ROW_VALUES;
        double sum[2];
        float b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int t = 2 * lane + e;
            const int64_t index = (row + t) * shape.heads + head;
            const double step = t < count ? double(gate(g, index, shape.gates_bf16)) * 1.4426950408889634 : 0.;
            sum[e] = step < -256. ? -256. : step;
            b[e] = t < count ? gate(beta, index, shape.gates_bf16) : 0.f;
        }
        sum[1] += sum[0];
        double before = sum[1];
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const double other = __shfl_up_sync(FULL, before, s);
            if (lane >= s) before += other;
        }
        const double total = __shfl_sync(FULL, before, 31);
        before -= sum[1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int t = 2 * lane + e;
            const double here = before + sum[e];
            const float hi = float(here), lo = float(here - double(hi));
            table[t] = hi, table[CHUNK + t] = lo, table[2 * CHUNK + t] = b[e];
            const float tail = ex2(float(total - here));
            rows[ROW_DECAY + t] = ex2(hi) * (1.f + lo * .6931471805599453f);
            rows[ROW_BETA + t] = b[e];
            rows[ROW_TAIL + t] = tail;
            rows[ROW_WRITE + t] = b[e] * tail;
            rows[ROW_HIGH + t] = hi;
            rows[ROW_LOW + t] = lo;
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    // K K^T and Q K^T: warp w takes rows 16 w .. 16 w + 15 and the column tiles up to the diagonal
    float kk[CHUNK / 8][4], qk[CHUNK / 8][4];
#pragma unroll
    for (int n = 0; n < CHUNK / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) kk[n][e] = qk[n][e] = 0.f;
    {
        const unsigned own = base + warp * 16 * PITCH + rows_first(lane, PITCH), own_q = own + CHUNK * PITCH;
        const unsigned all = base + cols_first(lane, PITCH);
#pragma unroll
        for (int kb = 0; kb < D / 16; ++kb) {
            unsigned ka[4], qa[4];
            ldsm4(ka, own + kb * 32);
            ldsm4(qa, own_q + kb * 32);
#pragma unroll
            for (int np = 0; np < CHUNK / 16; ++np) {
                if (np > warp) continue;
                unsigned b[4];
                ldsm4(b, all + np * 16 * PITCH + kb * 32);
                mma16816(kk[2 * np], ka, b[0], b[1]);
                mma16816(kk[2 * np + 1], ka, b[2], b[3]);
                mma16816(qk[2 * np], qa, b[0], b[1]);
                mma16816(qk[2 * np + 1], qa, b[2], b[3]);
            }
        }
    }
    __syncthreads();  // K and Q have been read: their room takes A and T
    const unsigned a = base, t = base + 2 * SQUARE;
    float* diagonal = reinterpret_cast<float*>(shared + Shared::DIAGONALS) + warp * 16 * DIAGONAL;
    {
        unsigned* p = reinterpret_cast<unsigned*>(saved.p + place * MATRIX);
#pragma unroll
        for (int n = 0; n < CHUNK / 8; ++n) {
            if (n > 2 * warp + 1) continue;
            const int s = 8 * n + 2 * (lane & 3);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int i = 16 * warp + 8 * half + (lane >> 2);
                float pv[2], av[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float between = ex2((table[i] - table[s + e]) + (table[CHUNK + i] - table[CHUNK + s + e]));
                    pv[e] = s + e <= i ? shape.scale * between * qk[n][2 * half + e] : 0.f;
                    av[e] = s + e < i ? between * kk[n][2 * half + e] * table[2 * CHUNK + s + e] : 0.f;
                }
                p[tile_at(warp, n >> 1) / 4 + (2 * half + (n & 1)) * 32 + lane] = pack2(pv[0], pv[1]);
                if (n >> 1 == warp) {
                    *reinterpret_cast<float2*>(diagonal + (i & 15) * DIAGONAL + (s & 15)) = make_float2(av[0], av[1]);
                } else {
                    const unsigned value = pack2(av[0], av[1]);
                    *reinterpret_cast<unsigned*>(shared + i * SQUARE_PITCH + s * 2) = value;
                    *reinterpret_cast<unsigned*>(shared + SQUARE + i * SQUARE_PITCH + s * 2) = pack2_rest(av[0], av[1], value);
                }
            }
        }
    }
    __syncwarp();
    {
        // the warp's diagonal tile: lane j (both halves of the warp alike) holds column j of its inverse
        const int j = lane & 15;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float sum0 = i == j ? 1.f : 0.f, sum1 = 0.f;
#pragma unroll
            for (int s = 0; s < i; s += 4) {
                const float4 c = *reinterpret_cast<const float4*>(diagonal + i * DIAGONAL + s);  // zero from the diagonal on
                sum0 -= c.x * x[s];
                if (s + 1 < i) sum1 -= c.y * x[s + 1];
                if (s + 2 < i) sum0 -= c.z * x[s + 2];
                if (s + 3 < i) sum1 -= c.w * x[s + 3];
            }
            x[i] = sum0 + sum1;
        }
        // the lower half of the lanes writes the values, the upper one the remainders
        __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(shared + 2 * SQUARE + (lane < 16 ? 0 : SQUARE)) + 16 * warp + j;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const __nv_bfloat16 value = __float2bfloat16(x[i]);
            to[(16 * warp + i) * (SQUARE_PITCH / 2)] = lane < 16 ? value : __float2bfloat16(x[i] - bf2f(value));
        }
        // the tile right of it lies above the diagonal and is read as a part of T2
        if (!(warp & 1)) {
            *reinterpret_cast<uint4*>(shared + 2 * SQUARE + (16 * warp + (lane >> 1)) * SQUARE_PITCH + (16 * warp + 16) * 2 + (lane & 1) * 16) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(shared + 3 * SQUARE + (16 * warp + (lane >> 1)) * SQUARE_PITCH + (16 * warp + 16) * 2 + (lane & 1) * 16) = make_uint4(0, 0, 0, 0);
        }
    }
    __syncthreads();
    if (warp < 2) join<16, 1>(a, t, 32 * warp, 0, 0, lane);
    __syncthreads();
    join<32, 1>(a, t, 0, 16 * (warp & 1), warp >> 1, lane);
    __syncthreads();
    for (int i = thread; i < MATRIX / 8; i += PREPARE_THREADS) {
        const int tile = i >> 5, block = (i >> 3) & 3, r = i & 7;
        const int rt = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, ct = tile - rt * (rt + 1) / 2;
        const int from = 2 * SQUARE + (16 * rt + 8 * (block >> 1) + r) * SQUARE_PITCH + (16 * ct + 8 * (block & 1)) * 2;
        reinterpret_cast<uint4*>(saved.t + place * MATRIX)[i] = *reinterpret_cast<const uint4*>(shared + from);
        if (saved.t_rest) reinterpret_cast<uint4*>(saved.t_rest + place * MATRIX)[i] = *reinterpret_cast<const uint4*>(shared + from + SQUARE);
    }
}

template <int D>
cudaError_t launch(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const void* g, const void* beta,
                   const DeltaSaved& saved, cudaStream_t stream) {
    constexpr int BYTES = PrepareShared<D>::BYTES;
    if (cudaError_t status = allow_shared<delta_prepare_kernel<D>>(BYTES)) return status;
    KernelTimer timer("delta_prepare", stream);
    delta_prepare_kernel<D><<<dim3(unsigned(shape.layout.slots()), shape.heads), PREPARE_THREADS, BYTES, stream>>>(shape, q, k, g, beta, saved);
    return cudaGetLastError();
}
}  // namespace

cudaError_t launch_delta_prepare(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const void* g,
                                 const void* beta, const DeltaSaved& saved, cudaStream_t stream) {
    if (shape.d == 32) return launch<32>(shape, q, k, g, beta, saved, stream);
    if (shape.d == 64) return launch<64>(shape, q, k, g, beta, saved, stream);
    return launch<128>(shape, q, k, g, beta, saved, stream);
}

}  // namespace dism
