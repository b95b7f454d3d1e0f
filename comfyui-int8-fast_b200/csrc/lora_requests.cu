// Low-rank adapters of many requests beside one shared int8 projection: row m of the batch belongs to a request whose
// adapter is a(m) (or to none), and
//
//   t[m]  = round(x[m] . A_a(m)^T)                   A_a [r, K], one slice of a bank [n, r, K]
//   y[m]  = base[m] + t[m] . B_a(m)^T                B_a [N, r], one slice of a bank [n, N, r]
//
// t is rounded to the 16-bit type of x (as in the single-adapter path, whose second product takes 16-bit operands); all
// sums are fp32.
//
// The batch is cut into tiles of 256 rows.  A tile with few adapters runs on the tensor cores: the MMAs of each of its
// adapters update only the rows (tensor-memory lanes) that use it, so the x tile is staged once whatever the adapters, and
// neither an adapter nor a row can reach what belongs to another.  Tiles where single tokens of many adapters meet arrive
// as CHUNKS instead, at most four consecutive rows with one adapter, whose factors ordinary warps read once per chunk.
// An MMA costs a tile the same for one row as for all, so in the down projection (one per adapter and 64 columns of K) an
// adapter's few rows beside others are chunks too; the up projection (one per adapter and 64 ranks) keeps them on the tensor
// cores.  1531 rows, K = N = 4096, rank 64: all adapters of a tile on the tensor cores, at most 8 of them: 80 us; their few
// rows as chunks: 72 us; then up to 16 adapters a tile, 8 of them with more rows: 60 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.h"
#include "low_rank.cuh"
#include "ptx_sm100.cuh"
#include "tensor_maps.h"

namespace i8f {
namespace {

constexpr int kChunkRows = kLowRankRows;

static_assert(sizeof(RequestTile) == 16 && sizeof(RequestSlot) == 48, "layout of the plan's tables");

template <int DT>
__device__ __forceinline__ void store_dt(void* out, int64_t idx, float v) {
    if constexpr (DT == I8F_BF16) static_cast<__nv_bfloat16*>(out)[idx] = __float2bfloat16_rn(v);
    else static_cast<__half*>(out)[idx] = __float2half_rn(v);
}

// ------------------------------------------------------------------ chunks: ordinary warps
// t of one chunk for RB rank rows of its adapter, by a CTA: every thread takes the same eight columns of the chunk's rows of x
// and of the RB rows of A, 256 threads side by side, so a CTA's share of A is in flight at once.  Bound by the bytes of A and,
// for few chunks, by one trip to memory; x is read again by the other rank rows' CTAs from L2.  A chunk without an
// adapter gets zeros.
// QUANT: the CTAs of a chunk also turn its rows into int8, dealt out over the rank rows (the arithmetic of i8f_quant_rowwise:
// step = max(absmax / 127, 1e-30), rint(x * (1 / step))), which saves a small batch a launch of its own for that.
constexpr int kChunkThreads = 256;
constexpr int kChunkWarps = kChunkThreads / 32;

struct QuantOut {
    int8_t* q;
    int64_t ldq;
    float* scale;
};

template <int DT, int RB, bool QUANT>
__global__ void __launch_bounds__(kChunkThreads)
down_chunks_kernel(const void* __restrict__ x, int64_t ldx, const void* __restrict__ bank_a, int K, int r,
                   const int4* __restrict__ chunks, void* __restrict__ t, int64_t ldt, const QuantOut out, int wait_first) {
    constexpr int kValues = RB * kChunkRows;
    __shared__ float s_part[kChunkWarps][kValues];
    __shared__ uint32_t s_max[kChunkWarps];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (wait_first) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 c = chunks[blockIdx.x];      // first row, rows, adapter
    const int j0 = blockIdx.y * RB;
    const int nvec = K >> 3;
    const uint16_t* const x0 = static_cast<const uint16_t*>(x) + c.x * ldx;
    if constexpr (QUANT) {
        for (int m = blockIdx.y; m < c.y; m += gridDim.y) {
            const uint4* const xr = reinterpret_cast<const uint4*>(x0 + m * ldx);
            // 16-bit patterns without their sign order like the values
            uint32_t m2 = 0u;
#pragma unroll 2
            for (int v = threadIdx.x; v < nvec; v += kChunkThreads) {
                const uint4 w = __ldg(xr + v);
                m2 = __vmaxu2(__vmaxu2(__vmaxu2(m2, w.x & 0x7FFF7FFFu), __vmaxu2(w.y & 0x7FFF7FFFu, w.z & 0x7FFF7FFFu)), w.w & 0x7FFF7FFFu);
            }
            uint32_t big = __reduce_max_sync(0xFFFFFFFFu, max(m2 & 0xFFFFu, m2 >> 16));
            if (lane == 0) s_max[warp] = big;
            __syncthreads();
            big = s_max[0];
#pragma unroll
            for (int w = 1; w < kChunkWarps; ++w) big = max(big, s_max[w]);
            __syncthreads();      // before the next row's
            const float amax = DT == I8F_BF16 ? __uint_as_float(big << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(big)));
            float step = __fdiv_rn(amax, 127.0f);
            if (step < 1e-30f) step = 1e-30f;      // not by fmaxf: a NaN stays in the step and makes the row NaN
            const float inv = __fdiv_rn(1.0f, step);
            const int64_t row = static_cast<int64_t>(c.x) + m;
            if (threadIdx.x == 0) out.scale[row] = step;
            constexpr float kMagic = 12582912.0f;      // 1.5 * 2^23
#pragma unroll 2
            for (int v = threadIdx.x; v < nvec; v += kChunkThreads) {
                float f[8];
                uint32_t u[8];
                widen8<DT == I8F_BF16>(__ldg(xr + v), f);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(__fadd_rn(__fmul_rn(f[e], inv), kMagic)) & 0xFFu;
                *reinterpret_cast<uint2*>(out.q + row * out.ldq + v * 8) =
                    make_uint2(u[0] | (u[1] << 8) | (u[2] << 16) | (u[3] << 24), u[4] | (u[5] << 8) | (u[6] << 16) | (u[7] << 24));
            }
        }
    }
    if (c.z >= 0) {
        float acc[RB][kChunkRows];
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int m = 0; m < kChunkRows; ++m) acc[j][m] = 0.f;
        const uint4* const a = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(bank_a) + (static_cast<int64_t>(c.z) * r + j0) * K);
#pragma unroll 2
        for (int v = threadIdx.x; v < nvec; v += kChunkThreads) {
            uint4 ra[RB], rx[kChunkRows];
#pragma unroll
            for (int j = 0; j < RB; ++j) ra[j] = __ldg(a + static_cast<int64_t>(j) * nvec + v);
#pragma unroll
            for (int m = 0; m < kChunkRows; ++m)
                rx[m] = m < c.y ? __ldg(reinterpret_cast<const uint4*>(x0 + m * ldx) + v) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int m = 0; m < kChunkRows; ++m) {
                if (m < c.y) {
                    float fx[8];
                    widen8<DT == I8F_BF16>(rx[m], fx);
#pragma unroll
                    for (int j = 0; j < RB; ++j) {
                        float fa[8];
                        widen8<DT == I8F_BF16>(ra[j], fa);
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[j][m] = fmaf(fx[e], fa[e], acc[j][m]);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < RB; ++j) {
#pragma unroll
            for (int m = 0; m < kChunkRows; ++m) {
                if (m < c.y) {
#pragma unroll
                    for (int d = 16; d; d >>= 1) acc[j][m] += __shfl_xor_sync(0xFFFFFFFFu, acc[j][m], d);
                    if (lane == 0) s_part[warp][j * kChunkRows + m] = acc[j][m];
                }
            }
        }
    }
    __syncthreads();
    if (threadIdx.x < kValues) {
        const int j = threadIdx.x / kChunkRows, m = threadIdx.x % kChunkRows;
        if (m < c.y) {
            float v = 0.f;
            if (c.z >= 0)
                for (int w = 0; w < kChunkWarps; ++w) v += s_part[w][threadIdx.x];
            store_dt<DT>(t, (static_cast<int64_t>(c.x) + m) * ldt + j0 + j, v);
        }
    }
    // this kernel's completion implies that of the one it may have run beside
    if (!wait_first && threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The up projection of the chunks into the fp32 addend of the int8 product's epilogue: one warp per (chunk, 64 columns).
// Bound by the bytes of B.  Rows without an adapter are not written.
constexpr int kUpCols = 64;
template <int DT>
__global__ void __launch_bounds__(128)
up_chunks_kernel(const void* __restrict__ t, int64_t ldt, const void* __restrict__ bank_b, int N, int r,
                 const int4* __restrict__ chunks, float* __restrict__ addend, int64_t ld_addend) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 c = chunks[blockIdx.x];      // first row, rows, adapter, first row in the addend
    const int n0 = (blockIdx.y * 4 + (threadIdx.x >> 5)) * kUpCols;
    if (c.z < 0 || c.w < 0 || n0 >= N) return;
    const uint16_t* const b[1] = {static_cast<const uint16_t*>(bank_b) + (static_cast<int64_t>(c.z) * N + n0) * r};
    low_rank_rows<DT == I8F_BF16, 1, 4>(static_cast<const uint16_t*>(t) + c.x * ldt, ldt, {0}, {c.y}, b, min(kUpCols, N - n0), r,
                                        addend + static_cast<int64_t>(c.w) * ld_addend + n0, ld_addend, threadIdx.x & 31);
}

// ------------------------------------------------------------------ down projection on the tensor cores
// t of one 128-row block: D [128, bn] in tensor memory += x slab [128, 64] . A_a slab [bn, 64]^T for every adapter a of the
// block, under a's row mask.  x is read once; 18432 x 4096 with four adapters of rank 32 takes 30 us = 5.0 TB/s.  A cluster of up to eight CTAs splits K where there
// are fewer blocks than SMs; its partial sums meet through distributed shared memory, every CTA adding its share of the
// rows in rank order (the same bits every time).
// Two rings: x slabs (one per K step) and adapter slabs (one per K step and adapter).
constexpr int kDownRows = 128;
constexpr int kDownThreads = 192;
// Up to rank 128 the rings take 96 KB, so that two CTAs share an SM: clusters of four or eight whole SMs do not fill the GPU's
// groups of SMs (4608 rows, K 4096, rank 64, clusters of four with one CTA per SM: 26.1 us in two waves).
constexpr int kAStages = 4;
constexpr int kASlab = kDownRows * 128;
constexpr int kMaxBStages = 8;
constexpr int kMaxBN = 256;
__host__ __device__ constexpr int b_ring_bytes(int bn) { return bn <= 128 ? 32 * 1024 : 64 * 1024; }
__host__ __device__ constexpr int b_ring_stages(int bn) {
    return b_ring_bytes(bn) / (bn * 128) < kMaxBStages ? b_ring_bytes(bn) / (bn * 128) : kMaxBStages;
}
constexpr int down_smem(int bn) { return kAStages * kASlab + b_ring_bytes(bn) + 1024 /* barriers */ + 1024 /* alignment */; }
static_assert(b_ring_stages(kMaxBN) >= 2 && b_ring_stages(128) >= 2, "a slab in use and one on its way");
static_assert(kDownRows * kMaxBN * 4 <= kAStages * kASlab + b_ring_bytes(kMaxBN) && kDownRows * 128 * 4 <= kAStages * kASlab + b_ring_bytes(128),
              "the partial sums land where the rings were");

enum : int { kStDownEmptyA = 121, kStDownEmptyB = 122, kStDownFullA = 123, kStDownFullB = 124, kStDownDone = 125 };

struct DownParams {
    int M, r, bn, b_stages, num_kb, split, bf16, wait_first;
    const RequestTile* tiles;
    const RequestSlot* slots;
    const int* row_adapter;
    void* t;
    int64_t ldt;
    int* status;
};

__global__ void __launch_bounds__(kDownThreads, 2)
down_tiles_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_a, const DownParams p) {
    const int block = blockIdx.y;
    const int half = block & 1;
    const RequestTile tile = p.tiles[block >> 1];
    if (tile.addend_row >= 0) return;            // a chunked tile; the whole cluster leaves
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen_base = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t a_ring = smem_base, b_ring = smem_base + kAStages * kASlab;
    const uint32_t b_slab = static_cast<uint32_t>(p.bn) * 128u;
    const uint32_t full_a = smem_base + kAStages * kASlab + b_ring_bytes(p.bn), empty_a = full_a + 8 * kAStages, full_b = empty_a + 8 * kAStages,
                   empty_b = full_b + 8 * kMaxBStages, done = empty_b + 8 * kMaxBStages, tmem_slot = done + 8;
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(gen_base + (tmem_slot - smem_base));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen_base + (tmem_slot - smem_base) + 4);
    volatile int* slot_count = abort_flag + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int n0 = static_cast<int>(blockIdx.z) * p.bn;
    // the block's adapters and the complement of their rows (what their MMAs leave alone)
    __shared__ int s_adapter[kMaxTileSlots];
    __shared__ uint32_t s_off[kMaxTileSlots][4];
    __shared__ uint32_t s_rows[4];      // the rows that the block works out; those of its other adapters are left to the chunks
    if (warp == 2) {
        bool mine = false;
        int adapter = 0;
        uint32_t off[4] = {};
        if (lane < tile.n_slots) {
            const RequestSlot& slot = p.slots[tile.slot_begin + lane];
            adapter = slot.adapter;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                off[i] = ~slot.rows[4 * half + i];
                mine |= off[i] != 0xFFFFFFFFu;
            }
            mine = mine && slot.few == 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t all = __reduce_or_sync(0xFFFFFFFFu, mine ? ~off[i] : 0u);
            if (lane == 0) s_rows[i] = all;
        }
        const uint32_t with_rows = __ballot_sync(0xFFFFFFFFu, mine);
        if (mine) {
            const int at = __popc(with_rows & ((1u << lane) - 1u));
            s_adapter[at] = adapter;
#pragma unroll
            for (int i = 0; i < 4; ++i) s_off[at][i] = off[i];
        }
        if (lane == 0) *slot_count = __popc(with_rows);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * kAStages + 2 * kMaxBStages + 1; ++i) mbar_init(full_a + 8 * i, 1);
        *abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_a);
    }
    if (warp == 1) tmem_alloc<kMaxBN>(tmem_slot);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot_ptr;
    // x may come from the kernel before this one only when the caller says so; where it does not, the whole pass runs beside
    // that kernel's tail, and the wait at the end makes this kernel's completion imply the other's
    if (p.wait_first) asm volatile("griddepcontrol.wait;" ::: "memory");

    const int kb0 = p.num_kb * rank / p.split, kb1 = p.num_kb * (rank + 1) / p.split;
    const int n_slots = *slot_count;
    const bool any = n_slots > 0;
    if (any && warp == 0 && lane == 0) {
        int sa = 0, sb = 0;
        uint32_t pa = 0, pb = 0;
        bool ok = true;
        for (int kb = kb0; ok && kb < kb1; ++kb) {
            if (!mbar_wait_bounded(empty_a + 8 * sa, pa ^ 1u, abort_flag, p.status, kStDownEmptyA)) break;
            mbar_arrive_expect_tx(full_a + 8 * sa, kASlab);
            tma_load_2d(a_ring + sa * kASlab, &tm_x, full_a + 8 * sa, kb * 64, block * kDownRows);
            if (++sa == kAStages) {
                sa = 0;
                pa ^= 1u;
            }
            for (int s = 0; s < n_slots; ++s) {
                if (!mbar_wait_bounded(empty_b + 8 * sb, pb ^ 1u, abort_flag, p.status, kStDownEmptyB)) {
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(full_b + 8 * sb, b_slab);
                tma_load_2d(b_ring + sb * b_slab, &tm_a, full_b + 8 * sb, kb * 64, s_adapter[s] * p.r + n0);
                if (++sb == p.b_stages) {
                    sb = 0;
                    pb ^= 1u;
                }
            }
        }
    } else if (any && warp == 1 && lane == 0) {
        int sa = 0, sb = 0;
        uint32_t pa = 0, pb = 0;
        bool ok = true;
        const uint32_t fmt = p.bf16 ? kFmtBF16 : kFmtF16;
        const uint32_t idesc = make_idesc(kDFmtF32, fmt, kDownRows, static_cast<uint32_t>(p.bn));
        for (int kb = kb0; ok && kb < kb1; ++kb) {
            if (!mbar_wait_bounded(full_a + 8 * sa, pa, abort_flag, p.status, kStDownFullA)) break;
            const uint64_t adesc = make_smem_desc_sw128(a_ring + sa * kASlab);
            for (int s = 0; s < n_slots; ++s) {
                const uint32_t off[4] = {s_off[s][0], s_off[s][1], s_off[s][2], s_off[s][3]};
                if (!mbar_wait_bounded(full_b + 8 * sb, pb, abort_flag, p.status, kStDownFullB)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const uint64_t bdesc = make_smem_desc_sw128(b_ring + sb * b_slab);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16_masked(tmem, adesc + 2 * k, bdesc + 2 * k, idesc, (kb != kb0 || k != 0) ? 1u : 0u, off);
                mma_commit(empty_b + 8 * sb);
                if (++sb == p.b_stages) {
                    sb = 0;
                    pb ^= 1u;
                }
            }
            if (!ok) break;
            mma_commit(empty_a + 8 * sa);
            if (++sa == kAStages) {
                sa = 0;
                pa ^= 1u;
            }
        }
        if (ok) mma_commit(done);
    }
    __syncwarp();

    const int quarter = warp & 3;
    const int row_in_block = quarter * 32 + lane;
    const int64_t row = static_cast<int64_t>(block) * kDownRows + row_in_block;
    const int cols = min(p.bn, p.r - n0);
    auto pack = [&](float lo, float hi) -> uint32_t {
        if (p.bf16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
            return *reinterpret_cast<const uint32_t*>(&h);
        }
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    };
    if (warp >= 2) {
        if (any) mbar_wait_bounded(done, 0, abort_flag, p.status, kStDownDone);
        tc_fence_after_sync();
    }
    if (p.split > 1) {
        // every CTA's MMAs are done: the rings are free, and each CTA sends every other its rows of the partial sums,
        // [source][column][row]: the lanes of a remote store are neighbours
        cluster_arrive();
        cluster_wait();
        const int share = kDownRows / p.split;
        if (warp >= 2 && any) {
            const uint32_t dst = mapa_cluster(smem_base, static_cast<uint32_t>(row_in_block / share)) +
                                 static_cast<uint32_t>((rank * p.bn * share + row_in_block % share) * 4);
            for (int c = 0; c < p.bn; c += 16) {
                uint32_t v[16];
                tmem_ld_32x16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(dst + static_cast<uint32_t>((c + j) * share * 4)), "r"(v[j]) : "memory");
            }
        }
        cluster_arrive();
        cluster_wait();
        const float* part = reinterpret_cast<const float*>(gen_base);
        for (int i = threadIdx.x; i < share * (cols / 8); i += kDownThreads) {      // eight columns of one row; cols is a multiple of 8
            const int rl = i & (share - 1), c = i / share * 8;
            const int64_t m = static_cast<int64_t>(block) * kDownRows + rank * share + rl;
            if (m >= p.M) continue;
            const int rb = rank * share + rl;      // row of the block
            const bool here = (s_rows[rb >> 5] >> (rb & 31)) & 1u;
            if (!here && p.row_adapter[m] >= 0) continue;      // a chunk's row
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (here) {
                for (int src = 0; src < p.split; ++src) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += part[(src * p.bn + c + j) * share + rl];
                }
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.t) + m * p.ldt + n0 + c) =
                make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7]));
        }
    } else if (warp >= 2) {
        const bool use = (s_rows[quarter] >> lane) & 1u;
        const bool write = row < p.M && (use || p.row_adapter[row] < 0);
        for (int c = 0; c < cols; c += 16) {
            uint32_t v[16];
            tmem_ld_32x16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
            tmem_ld_wait();
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o[j] = pack(use ? __uint_as_float(v[2 * j]) : 0.f, use ? __uint_as_float(v[2 * j + 1]) : 0.f);
            }
            if (write) {      // cols is a multiple of 8
                uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.t) + row * p.ldt + n0 + c);
                dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
                if (c + 8 < cols) dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
            }
        }
    }
    if (!p.wait_first && threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag)      // copies still in flight get time to land before the CTA exits
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<kMaxBN>(tmem);
    }
}

// Whether the batch has tiles for the tensor cores / chunks for the warps / chunks whose up projection is theirs, too.
bool has_dense(const i8f_request_rows* rows) { return rows->n_dense > 0; }
bool has_chunks(const i8f_request_rows* rows) { return rows->n_chunks > 0; }
bool has_addend(const i8f_request_rows* rows) { return rows->addend_rows > 0; }

int check_rows(const i8f_request_rows* rows, int64_t M) {
    I8F_REQUIRE(rows != nullptr, I8F_ERR_INVALID_ARG, "rows is NULL");
    I8F_REQUIRE(rows->rows == M && M < (1LL << 31) - 256, I8F_ERR_INVALID_ARG, "the row plan is for %lld rows, the call has %lld",
                (long long)rows->rows, (long long)M);
    I8F_REQUIRE(M == 0 || (rows->row_adapter != nullptr && rows->n_dense >= 0 && rows->n_chunks >= 0 && rows->n_dense + rows->n_chunks > 0 &&
                           (rows->n_chunks == 0 || rows->chunks != nullptr) &&
                           (rows->n_dense == 0 || (rows->tiles != nullptr && rows->slots != nullptr)) &&
                           rows->addend_rows >= 0 && (rows->n_dense > 0 || rows->addend_rows > 0)),
                I8F_ERR_INVALID_ARG, "incomplete row plan");
    return I8F_OK;
}

int check_bank(const void* bank, int64_t adapters, int64_t r, const i8f_request_rows* rows, int dtype, const char* what) {
    I8F_REQUIRE(dtype == I8F_BF16 || dtype == I8F_F16, I8F_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", what);
    I8F_REQUIRE(bank != nullptr && adapters > 0 && adapters > rows->max_adapter, I8F_ERR_INVALID_ARG,
                "%s: the rows name adapter %d, the bank has %lld", what, rows->max_adapter, (long long)adapters);
    I8F_REQUIRE(r > 0 && r % 8 == 0 && r <= 1024, I8F_ERR_UNSUPPORTED, "%s: the rank %lld must be a multiple of 8, at most 1024", what,
                (long long)r);
    I8F_REQUIRE(aligned16(bank), I8F_ERR_ALIGNMENT, "%s: the bank must be 16-byte aligned", what);
    return I8F_OK;
}

int64_t addend_pitch(int64_t N) { return (N + 31) / 32 * 32; }
size_t padded(size_t bytes) { return (bytes + 255) & ~size_t(255); }
size_t addend_bytes(const i8f_request_rows* rows, int64_t N) {
    return static_cast<size_t>(rows->addend_rows) * static_cast<size_t>(addend_pitch(N)) * sizeof(float);
}

int check_down(const void* x, int64_t ldx, const void* bank_a, int64_t adapters, int64_t r, const i8f_request_rows* rows, const void* t,
               int64_t ldt, int dtype, int64_t K) {
    int rc = check_bank(bank_a, adapters, r, rows, dtype, "bank_a");
    if (rc != I8F_OK) return rc;
    I8F_REQUIRE(x != nullptr && t != nullptr && ldx >= K && ldt >= r && K > 0, I8F_ERR_INVALID_ARG, "bad x or t");
    I8F_REQUIRE(aligned16(x) && aligned16(t) && K % 8 == 0 && ldx % 8 == 0 && ldt % 8 == 0, I8F_ERR_ALIGNMENT,
                "x and t must be 16-byte aligned, K and both pitches multiples of 8 elements");
    I8F_REQUIRE(K < (1LL << 31) - 256 && adapters * r < (1LL << 31), I8F_ERR_UNSUPPORTED, "dimension too large");
    return I8F_OK;
}

int check_up(const void* t, int64_t ldt, const void* bank_b, int64_t adapters, int64_t r, const i8f_request_rows* rows, int dtype, int64_t N) {
    int rc = check_bank(bank_b, adapters, r, rows, dtype, "bank_b");
    if (rc != I8F_OK) return rc;
    I8F_REQUIRE(t != nullptr && ldt >= r, I8F_ERR_INVALID_ARG, "bad t");
    I8F_REQUIRE(aligned16(t) && ldt % 8 == 0, I8F_ERR_ALIGNMENT, "t must be 16-byte aligned, its pitch a multiple of 8 elements");
    I8F_REQUIRE(N <= 65535LL * 128 && adapters * N < (1LL << 31) - 512, I8F_ERR_UNSUPPORTED, "N=%lld is too large", (long long)N);
    return I8F_OK;
}

// The down projection of the dense tiles.  `after_reader`: the kernel before this one in the stream only reads what this one
// reads (it does not produce x), so the two may overlap.
int launch_down_tiles(const void* x, int64_t ldx, const void* bank_a, int64_t adapters, int64_t r, const i8f_request_rows* rows, void* t,
                      int64_t ldt, int dtype, int64_t M, int64_t K, bool after_reader, cudaStream_t st) {
    DownParams p{};
    p.M = static_cast<int>(M);
    p.r = static_cast<int>(r);
    p.bn = r >= kMaxBN ? kMaxBN : static_cast<int>((r + 15) / 16 * 16);
    p.b_stages = b_ring_stages(p.bn);
    p.num_kb = static_cast<int>((K + 63) / 64);
    p.bf16 = dtype == I8F_BF16;
    p.wait_first = after_reader ? 0 : 1;
    p.tiles = reinterpret_cast<const RequestTile*>(rows->tiles);
    p.slots = reinterpret_cast<const RequestSlot*>(rows->slots);
    p.row_adapter = rows->row_adapter;
    p.t = t;
    p.ldt = ldt;
    p.status = device_status_word();
    I8F_REQUIRE(p.status != nullptr, I8F_ERR_CUDA, "device status word unavailable");
    CUtensorMap tm_x, tm_a;
    const int kind = p.bf16 ? kKindBF16 : kKindF16;
    int rc = make_operand_map(&tm_x, kind, x, M, K, ldx, kDownRows);
    if (rc != I8F_OK) return rc;
    rc = make_operand_map(&tm_a, kind, bank_a, adapters * r, K, K, p.bn);
    if (rc != I8F_OK) return rc;
    const int64_t blocks = (M + kDownRows - 1) / kDownRows, rank_tiles = (r + p.bn - 1) / p.bn;
    I8F_REQUIRE(blocks <= 65535, I8F_ERR_UNSUPPORTED, "M=%lld is too large", (long long)M);
    const int64_t dense = rows->n_dense * 2 < blocks ? rows->n_dense * 2 : blocks;
    p.split = 1;
    // CTAs that share a block's K range, with at least four slabs each.  A 128-row MMA takes 128 cycles however few columns it
    // has, so a block's K loop is bound by the tensor core of its SM (0.43 us per slab) and is spread over as many SMs as there
    // are (us at K 4096, split 1 / 2 / 4 / 8: 9216 rows 32.8 / 21.9 / 28.2 / 28.4, 4608 rows 32.2 / 21.0 / 15.1 / 21.1,
    // 1536 rows 31.4 / 19.9 / 12.7 / 10.2); two CTAs on every SM still gain a little (18432 rows: 34.3 / 30.3).
    while (p.split < 8 && dense * rank_tiles * p.split * 2 <= sm_count() && p.num_kb >= 8 * p.split) p.split *= 2;
    if (p.split == 1 && p.bn <= 128 && dense * rank_tiles <= sm_count() && p.num_kb >= 8) p.split = 2;
    static bool attr_done[64] = {false};
    const int dev = current_device();
    if (!attr_done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(down_tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, down_smem(kMaxBN));
        if (e != cudaSuccess) return fail(I8F_ERR_CUDA, "cudaFuncSetAttribute(smem=%d): %s", down_smem(kMaxBN), cudaGetErrorString(e));
        attr_done[dev] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.split), static_cast<unsigned>(blocks), static_cast<unsigned>(rank_tiles));
    cfg.blockDim = dim3(kDownThreads, 1, 1);
    cfg.dynamicSmemBytes = down_smem(p.bn);
    cfg.stream = st;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(p.split);
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, down_tiles_kernel, tm_x, tm_a, p);
    if (e != cudaSuccess) return fail(I8F_ERR_CUDA, "down_tiles_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("down_tiles_kernel");
}

// `out`: also quantise the rows (only where the chunks cover the whole batch).  `after_reader` as in launch_down_tiles, the kernels
// before it being the library's own.
int launch_down_chunks(const void* x, int64_t ldx, const void* bank_a, int64_t r, const i8f_request_rows* rows, void* t, int64_t ldt,
                       int dtype, int64_t K, const QuantOut* out, bool after_reader, cudaStream_t st) {
    const int4* chunks = reinterpret_cast<const int4*>(rows->chunks);
    // two rank rows per CTA where the chunks alone would leave SMs idle, else eight (x is then read a quarter as often)
    const bool few = rows->n_chunks * (r / 8) < 2 * sm_count();
    const dim3 grid(static_cast<unsigned>(rows->n_chunks), static_cast<unsigned>(r / (few ? 2 : 8)));
    const QuantOut q = out != nullptr ? *out : QuantOut{};
    const int k = static_cast<int>(K), rank = static_cast<int>(r);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kChunkThreads, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = after_reader ? 1 : 0;
    cudaError_t e = cudaSuccess;
#define I8F_DOWN(DT, RB, Q) e = cudaLaunchKernelEx(&cfg, down_chunks_kernel<DT, RB, Q>, x, ldx, bank_a, k, rank, chunks, t, ldt, q, after_reader ? 0 : 1)
#define I8F_DOWN_RB(DT)                                     \
    do {                                                    \
        if (few && out != nullptr) I8F_DOWN(DT, 2, true);   \
        else if (few) I8F_DOWN(DT, 2, false);               \
        else if (out != nullptr) I8F_DOWN(DT, 8, true);     \
        else I8F_DOWN(DT, 8, false);                        \
    } while (0)
    if (dtype == I8F_BF16) I8F_DOWN_RB(I8F_BF16);
    else I8F_DOWN_RB(I8F_F16);
#undef I8F_DOWN_RB
#undef I8F_DOWN
    if (e != cudaSuccess) return fail(I8F_ERR_CUDA, "down_chunks_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("down_chunks_kernel");
}

int launch_up_chunks(const void* t, int64_t ldt, const void* bank_b, int64_t r, const i8f_request_rows* rows, int dtype, int64_t N,
                     float* addend, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(rows->n_chunks), static_cast<unsigned>((N + 4 * kUpCols - 1) / (4 * kUpCols)));
    cfg.blockDim = dim3(128, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const int4* chunks = reinterpret_cast<const int4*>(rows->chunks);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, dtype == I8F_BF16 ? up_chunks_kernel<I8F_BF16> : up_chunks_kernel<I8F_F16>, t, ldt, bank_b,
                                             static_cast<int>(N), static_cast<int>(r), chunks, addend, addend_pitch(N));
    if (e != cudaSuccess) return fail(I8F_ERR_CUDA, "up_chunks_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("up_chunks_kernel");
}

int launch_down(const void* x, int64_t ldx, const void* bank_a, int64_t adapters, int64_t r, const i8f_request_rows* rows, void* t,
                int64_t ldt, int dtype, int64_t M, int64_t K, bool after_reader, cudaStream_t st) {
    if (has_dense(rows)) {
        const int rc = launch_down_tiles(x, ldx, bank_a, adapters, r, rows, t, ldt, dtype, M, K, after_reader, st);
        if (rc != I8F_OK) return rc;
    }
    return has_chunks(rows) ? launch_down_chunks(x, ldx, bank_a, r, rows, t, ldt, dtype, K, nullptr, after_reader, st) : I8F_OK;
}

RequestTerm request_term(const void* t, int64_t ldt, const void* bank_b, int64_t adapters, int64_t r, const i8f_request_rows* rows,
                         int64_t N, const float* addend) {
    RequestTerm term{};
    term.row_adapter = rows->row_adapter;
    term.addend = addend;
    term.ld_addend = addend_pitch(N);
    if (has_dense(rows)) {
        term.tiles = reinterpret_cast<const RequestTile*>(rows->tiles);
        term.slots = reinterpret_cast<const RequestSlot*>(rows->slots);
    }
    term.t = t;
    term.ldt = ldt;
    term.b = bank_b;
    term.adapters = adapters;
    term.r = r;
    return term;
}

}  // namespace
}  // namespace i8f

using namespace i8f;

extern "C" {

int i8f_lora_down_requests(const void* x, int64_t ldx, const void* bank_a, int64_t adapters, int64_t r, const i8f_request_rows* rows,
                           void* t, int64_t ldt, int dtype, int64_t M, int64_t K, void* stream) {
    int rc = check_rows(rows, M);
    if (rc != I8F_OK || M == 0) return rc;
    rc = check_down(x, ldx, bank_a, adapters, r, rows, t, ldt, dtype, K);
    if (rc != I8F_OK) return rc;
    return launch_down(x, ldx, bank_a, adapters, r, rows, t, ldt, dtype, M, K, false, static_cast<cudaStream_t>(stream));
}

size_t i8f_lora_requests_workspace_bytes(const i8f_request_rows* rows, int64_t N) {
    if (rows == nullptr || rows->rows <= 0 || N <= 0) return 0;
    return addend_bytes(rows, N);
}

int i8f_linear_w8a8_lora_requests(const int8_t* a, int64_t lda, const float* a_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                                  int w_scale_mode, const void* bias, int bias_dtype, const void* t, int64_t ldt, const void* bank_b,
                                  int64_t adapters, int64_t r, const i8f_request_rows* rows, void* out, int out_dtype, int64_t ldo,
                                  int64_t M, int64_t N, int64_t K, int epilogue_order, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    int rc = check_rows(rows, M);
    if (rc != I8F_OK || M == 0 || N == 0) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = check_up(t, ldt, bank_b, adapters, r, rows, out_dtype, N);
    if (rc != I8F_OK) return rc;
    const size_t need = addend_bytes(rows, N);
    I8F_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), I8F_ERR_WORKSPACE,
                "workspace too small: have %zu bytes, need %zu", workspace_bytes, need);
    I8F_REQUIRE(aligned16(workspace), I8F_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    float* addend = static_cast<float*>(workspace);
    const RequestTerm term = request_term(t, ldt, bank_b, adapters, r, rows, N, addend);
    for (const bool check_only : {true, false}) {     // everything is checked before anything is launched
        if (!check_only && has_addend(rows) && requests_need_addend(M, N, K)) {
            rc = launch_up_chunks(t, ldt, bank_b, r, rows, out_dtype, N, addend, st);
            if (rc != I8F_OK) return rc;
        }
        rc = linear_w8a8_requests(a, lda, a_scale, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, out_dtype, ldo, M, N, K,
                                  epilogue_order, term, check_only, st);
        if (rc != I8F_OK) return rc;
    }
    return I8F_OK;
}

// Workspace of the whole forward: int8 rows, their scales, the rotated rows (where the adapters see them), t, the addend (where
// the product reads one).
struct ForwardLayout {
    size_t scales, rotated, t, addend, total;
    ForwardLayout(const i8f_request_rows* rows, int64_t M, int64_t N, int64_t K, int64_t r, bool keep_rotated) {
        scales = padded(static_cast<size_t>(M) * K);
        rotated = scales + padded(static_cast<size_t>(M) * sizeof(float));
        t = rotated + (keep_rotated ? padded(static_cast<size_t>(M) * K * 2) : 0);
        addend = t + padded(static_cast<size_t>(M) * r * 2);
        total = addend + (requests_need_addend(M, N, K) ? addend_bytes(rows, N) : 0);
    }
};

size_t i8f_linear_lora_requests_workspace_bytes(const i8f_request_rows* rows, int64_t N, int64_t K, int64_t r, int hadamard128,
                                                int rotated_lora_input) {
    if (rows == nullptr || rows->rows <= 0 || N <= 0 || K <= 0 || r <= 0) return 0;
    return ForwardLayout(rows, rows->rows, N, K, r, hadamard128 && rotated_lora_input).total;
}

int i8f_linear_lora_requests(const void* x, int x_dtype, int64_t ldx, int hadamard128, int rotated_lora_input, const int8_t* w, int64_t ldw,
                             const float* w_scale, int w_scale_mode, const void* bias, int bias_dtype, const void* bank_a,
                             const void* bank_b, int64_t adapters, int64_t r, const i8f_request_rows* rows, void* out, int64_t ldo,
                             int64_t M, int64_t N, int64_t K, int epilogue_order, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_rows(rows, M);
    if (rc != I8F_OK || M == 0 || N == 0) return rc;
    I8F_REQUIRE(K > 0 && K % 16 == 0, I8F_ERR_ALIGNMENT, "K=%lld must be a multiple of 16", (long long)K);
    rc = check_bank(bank_a, adapters, r, rows, x_dtype, "bank_a");
    if (rc != I8F_OK) return rc;
    const bool keep_rotated = hadamard128 && rotated_lora_input;
    const ForwardLayout at(rows, M, N, K, r, keep_rotated);
    I8F_REQUIRE(workspace != nullptr && workspace_bytes >= at.total, I8F_ERR_WORKSPACE, "workspace too small: have %zu bytes, need %zu",
                workspace_bytes, at.total);
    I8F_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, I8F_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
    // the rotated copy has the pitch of its input in the quantiser
    I8F_REQUIRE(!keep_rotated || ldx == K, I8F_ERR_UNSUPPORTED, "rotated activations for the adapters need ldx == K");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int8_t* q = reinterpret_cast<int8_t*>(ws);
    float* q_scale = reinterpret_cast<float*>(ws + at.scales);
    void* rotated = keep_rotated ? ws + at.rotated : nullptr;
    void* t = ws + at.t;
    float* addend = reinterpret_cast<float*>(ws + at.addend);
    const void* lora_in = keep_rotated ? rotated : x;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = check_down(lora_in, ldx, bank_a, adapters, r, rows, t, r, x_dtype, K);
    if (rc != I8F_OK) return rc;
    rc = check_up(t, r, bank_b, adapters, r, rows, x_dtype, N);
    if (rc != I8F_OK) return rc;
    RequestTerm term = request_term(t, r, bank_b, adapters, r, rows, N, addend);
    term.after_own = true;
    rc = linear_w8a8_requests(q, K, q_scale, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, x_dtype, ldo, M, N, K, epilogue_order,
                              term, true, st);
    if (rc != I8F_OK) return rc;
    if (!has_dense(rows) && !hadamard128) {
        const QuantOut out_q{q, K, q_scale};
        rc = launch_down_chunks(x, ldx, bank_a, r, rows, t, r, x_dtype, K, &out_q, false, st);
    } else {
        rc = i8f_quant_rowwise(x, x_dtype, M, K, ldx, q, K, q_scale, hadamard128, rotated, stream);
        if (rc != I8F_OK) return rc;
        rc = launch_down(lora_in, ldx, bank_a, adapters, r, rows, t, r, x_dtype, M, K, !keep_rotated, st);
    }
    if (rc != I8F_OK) return rc;
    if (has_addend(rows) && requests_need_addend(M, N, K)) {
        rc = launch_up_chunks(t, r, bank_b, r, rows, x_dtype, N, addend, st);
        if (rc != I8F_OK) return rc;
    }
    return linear_w8a8_requests(q, K, q_scale, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, x_dtype, ldo, M, N, K, epilogue_order,
                                term, false, st);
}

size_t i8f_linear_w8a16_small_lora_requests_workspace_bytes(const i8f_request_rows* rows, int64_t N, int64_t r) {
    if (rows == nullptr || rows->rows <= 0 || N <= 0 || r <= 0) return 0;
    return static_cast<size_t>(rows->rows) * static_cast<size_t>(r) * 2;
}

int i8f_linear_w8a16_small_lora_requests(const void* x, int x_dtype, int64_t ldx, const int8_t* w, int64_t ldw, const float* w_scale,
                                         int w_scale_mode, const void* bias, int bias_dtype, const void* bank_a, const void* bank_b,
                                         int64_t adapters, int64_t r, const i8f_request_rows* rows, void* out, int64_t ldo, int64_t M,
                                         int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_rows(rows, M);
    if (rc != I8F_OK || M == 0 || N == 0) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const RequestTerm term = request_term(workspace, r, bank_b, adapters, r, rows, N, nullptr);
    rc = linear_small_requests(x, x_dtype, ldx, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, ldo, M, N, K, term, true, st);
    if (rc != I8F_OK) return rc;
    I8F_REQUIRE(!has_dense(rows), I8F_ERR_INVALID_ARG, "a row plan of at most 16 rows has chunks only");
    rc = check_bank(bank_a, adapters, r, rows, x_dtype, "bank_a");
    if (rc != I8F_OK) return rc;
    const size_t need = i8f_linear_w8a16_small_lora_requests_workspace_bytes(rows, N, r);
    I8F_REQUIRE(workspace != nullptr && workspace_bytes >= need, I8F_ERR_WORKSPACE, "workspace too small: have %zu bytes, need %zu",
                workspace_bytes, need);
    I8F_REQUIRE(aligned16(workspace), I8F_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    rc = check_down(x, ldx, bank_a, adapters, r, rows, workspace, r, x_dtype, K);
    if (rc != I8F_OK) return rc;
    rc = check_up(workspace, r, bank_b, adapters, r, rows, x_dtype, N);
    if (rc != I8F_OK) return rc;
    rc = launch_down_chunks(x, ldx, bank_a, r, rows, workspace, r, x_dtype, K, nullptr, false, st);
    if (rc != I8F_OK) return rc;
    return linear_small_requests(x, x_dtype, ldx, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, ldo, M, N, K, term, false, st);
}

}  // extern "C"
