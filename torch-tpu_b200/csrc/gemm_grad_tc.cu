// bf16 products of the gradients on the sm_100a tensor cores (tcgen05.mma kind::f16, fp32 accumulation in tensor memory):
//
//   weight gradient   C_g[m,n] = sum over the rows r of group g of  A[r,m] * B[r,n]
//                     the K axis is the rows (tokens): both operands lie MN-major in memory, a group's rows are a range
//                     that starts and ends anywhere.  Rows of experts: dW = d^T x.  One group: a linear layer's dW and the
//                     router's.
//   row product       C[r,n] = sum over k of  A[r,k] * B[k,n]     (A K-major, B MN-major): the router's dx
//
// One persistent CTA per SM, 8 warps: warp 0 = TMA producer, warp 1 = MMA issuer (and TMEM owner), warps 4..7 = epilogue
// (one lane quarter each).  A tile is 128 x 256 outputs; a K step is 64 deep: A 128 x 64 and B 64 x 256 (16 + 32 KB), four
// stages; two accumulators of 256 TMEM columns, so that the epilogue of a tile runs beside the next tile's MMAs.
// Results leave through swizzled shared-memory patches by TMA stores (or fp32 reductions), 32 rows x 128 bytes at a time.
//
// A group's last K step may reach past its end, into the next group's rows (or rows that nobody wrote): all of warp 1
// overwrites those rows of both operands with zeros before the MMAs read them - in the MN-major layout row r of a box is
// the 128 bytes at r * 128, so the tail is one contiguous run per box.
//
// The tensor cores' fp32 accumulation is not an IEEE one: against fp64 the error of a sum of K products grows with K (measured,
// random operands: 1e-6 of the result's norm at K = 1024, 4.4e-6 at 4096, 1.9e-5 at 16384).  fp32 results are therefore formed
// in pieces of kGradChunk rows that are added up in order in IEEE fp32: the first piece of a tile is stored (or added to
// what is there), the others added by the CTA that owns the tile, one after the other, so that equal calls give equal bits.
//
// Every wait is bounded; on a time-out status bit 1 is raised and all roles leave.
#include "tc_ptx.cuh"

namespace {

constexpr int GG_THREADS = 256;
constexpr int GG_STAGES = 4;
constexpr int GG_BK = 64;
constexpr int GG_A_BYTES = 128 * GG_BK * 2;  // 16 KB
constexpr int GG_B_BYTES = 256 * GG_BK * 2;  // 32 KB
constexpr int GG_STAGE_BYTES = GG_A_BYTES + GG_B_BYTES;
constexpr int GG_BOX_BYTES = GG_BK * 128;    // an MN-major box: 64 rows of K x 128 bytes
constexpr int GG_PATCH_BYTES = 32 * 128;
constexpr int kGradChunk = 2048;
static_assert(kGradChunk % GG_BK == 0, "pieces are whole K steps");

struct GgShared {
  uint64_t full[GG_STAGES], empty[GG_STAGES];
  uint64_t tmem_full[2], tmem_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr size_t GG_SMEM_BYTES = 1024 + (size_t)GG_STAGES * GG_STAGE_BYTES + 8 * GG_PATCH_BYTES + sizeof(GgShared);
static_assert(GG_SMEM_BYTES <= 232448, "more than the 227 KB of shared memory a CTA can have");

struct GgArgs {
  const int32_t* offsets;  // rows of group g: [offsets[g], offsets[g+1]); NULL = the `splits` even parts of [0, P)
  int P, groups, segs;     // segs: operand pairs that a group has (columns [seg * M, (seg + 1) * M) of A)
  int M, N, MT, NT;        // outputs of one (group, segment); tiles along both
  int out_rows;            // rows of the output between groups
  int K;                   // row product: depth; B's row of step k is k % kb_rows
  int kb_rows;
  int chunk;               // rows that one accumulator takes (0 = all)
  int out_f32, add;        // add: results are added to the output (fp32)
  int32_t* status;
};

// kind::f16, bf16 x bf16 -> fp32, M = 128, N = 256, B MN-major
__host__ __device__ constexpr uint32_t gg_idesc(int a_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn_major << 15) | (1u << 16) | ((256u >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void gg_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void gg_store(const CUtensorMap* map, int c0, int c1, uint32_t src, bool add) {
  if (add)
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(src)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(src)
                 : "memory");
}

// ROWS = false: weight gradient, true: row product
template <bool ROWS>
__global__ void __launch_bounds__(GG_THREADS, 1)
gemm_grad_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB0,
                 const __grid_constant__ CUtensorMap tmB1, const __grid_constant__ CUtensorMap tmC0,
                 const __grid_constant__ CUtensorMap tmC1, const __grid_constant__ CUtensorMap tmC2, const GgArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* patches = smem + (size_t)GG_STAGES * GG_STAGE_BYTES;
  GgShared* sh = reinterpret_cast<GgShared*>(patches + 8 * GG_PATCH_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem);
  volatile int* abort_flag = &sh->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < GG_STAGES; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sh->tmem_full[b]), 1);
      mbar_init(smem_u32(&sh->tmem_empty[b]), 4);
    }
    sh->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = sh->tmem_base;
  pdl_begin();

  const int per_group = a.segs * a.MT * a.NT, items = a.groups * per_group;
  struct Item {
    int g, seg, mt, nt, beg, end;  // rows of K [beg, end) (weight gradient)
  };
  // n-tile fastest: the CTAs that run together share a few m-tiles' columns of A and read all of B's
  auto item_of = [&](int t) {
    Item w;
    w.g = t / per_group;
    int r = t - w.g * per_group;
    w.seg = r / (a.MT * a.NT);
    r -= w.seg * a.MT * a.NT;
    w.mt = r / a.NT;
    w.nt = r - w.mt * a.NT;
    if (ROWS) {
      w.beg = 0, w.end = a.K;
    } else if (a.offsets) {
      w.beg = a.offsets[w.g];
      w.end = min(a.offsets[w.g + 1], a.P);
    } else {  // whole K steps to each part
      const int64_t steps = (a.P + GG_BK - 1) / GG_BK;
      w.beg = (int)(steps * w.g / a.groups) * GG_BK;
      w.end = min((int)(steps * (w.g + 1) / a.groups) * GG_BK, a.P);
    }
    return w;
  };
  auto piece = [&](const Item& w) { return a.chunk > 0 ? a.chunk : max(w.end - w.beg, 1); };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (one thread)
    if (lane == 0) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      Item nx{};
      if ((int)blockIdx.x < items) nx = item_of(blockIdx.x);
      for (int t = blockIdx.x; t < items && ok; t += gridDim.x) {
        const Item w = nx;
        if (t + (int)gridDim.x < items) nx = item_of(t + gridDim.x);  // its row range is on the way while this item loads
        const CUtensorMap* tmB = w.seg == 2 ? &tmB1 : &tmB0;
        const int m0 = w.seg * a.M + w.mt * 128, n0 = w.nt * 256;
        int brow = w.beg;
        for (int r = w.beg; r < w.end; r += GG_BK) {
          if (!mbar_wait(smem_u32(&sh->empty[0]) + s * 8, ph, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t full = smem_u32(&sh->full[0]) + s * 8, sa = smem_base + s * GG_STAGE_BYTES, sb = sa + GG_A_BYTES;
          mbar_arrive_expect_tx(full, GG_STAGE_BYTES);
          if (ROWS) {
            tma_load_2d(sa, &tmA, r, w.mt * 128, full);
          } else {
            tma_load_2d(sa, &tmA, m0, r, full);
            tma_load_2d(sa + GG_BOX_BYTES, &tmA, m0 + 64, r, full);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) tma_load_2d(sb + c * GG_BOX_BYTES, tmB, n0 + c * 64, brow, full);
          brow += GG_BK;
          if (ROWS && brow == a.kb_rows) brow = 0;
          if (++s == GG_STAGES) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (one thread; the warp clears tails)
    const uint32_t idesc = gg_idesc(ROWS ? 0 : 1);
    const uint64_t adesc0 = ROWS ? make_smem_desc(smem_base, 16, 1024) : make_smem_desc(smem_base, GG_BOX_BYTES, 1024);
    const uint64_t bdesc0 = make_smem_desc(smem_base + GG_A_BYTES, GG_BOX_BYTES, 1024);
    uint32_t s = 0, ph = 0, n = 0;
    bool ok = true;
    Item nx{};
    if ((int)blockIdx.x < items) nx = item_of(blockIdx.x);
    for (int t = blockIdx.x; t < items && ok; t += gridDim.x) {
      const Item w = nx;
      if (t + (int)gridDim.x < items) nx = item_of(t + gridDim.x);
      const int step = piece(w);
      for (int beg = w.beg; beg < w.end && ok; beg += step, ++n) {
        const int end = min(beg + step, w.end);
        const uint32_t buf = n & 1, d = tmem_base + buf * 256;
        // (one decision for the warp: its lanes stay together, also when a wait runs out)
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->tmem_empty[buf]), ((n >> 1) & 1) ^ 1, abort_flag))) {
          ok = false;
          break;
        }
        for (int r = beg; r < end; r += GG_BK) {
          if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->full[0]) + s * 8, ph, abort_flag))) {
            ok = false;
            break;
          }
          if (!ROWS && end - r < GG_BK) {  // the group ends inside this step: its other rows count as zeros
            const int from = (end - r) * 8, each = GG_BK * 8 - from;  // in 16-byte units of a box
            uint4* box = reinterpret_cast<uint4*>(smem + (size_t)s * GG_STAGE_BYTES);
            for (int i = lane; i < 6 * each; i += 32)
              box[(i / each) * (GG_BOX_BYTES / 16) + from + i % each] = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (lane == 0) {
            tc_fence_after();
            const uint64_t adesc = adesc0 + (uint64_t)(s * (GG_STAGE_BYTES >> 4)), bdesc = bdesc0 + (uint64_t)(s * (GG_STAGE_BYTES >> 4));
#pragma unroll
            for (int k16 = 0; k16 < GG_BK / 16; ++k16)  // +16 rows of 128 B (MN-major) or +32 B inside the swizzle atom (K-major)
              gg_mma(d, adesc + (uint64_t)(k16 * (ROWS ? 2 : 128)), bdesc + (uint64_t)(k16 * 128), idesc, (r > beg || k16 > 0) ? 1u : 0u);
            tc_commit(smem_u32(&sh->empty[0]) + s * 8);
          }
          if (++s == GG_STAGES) s = 0, ph ^= 1;
        }
        if (ok && lane == 0) tc_commit(smem_u32(&sh->tmem_full[buf]));
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue (4 warps, one lane quarter each)
    const int q = warp & 3;
    uint8_t* const patch0 = patches + q * (2 * GG_PATCH_BYTES);
    uint32_t n = 0;
    int stores = 0;
    bool ok = true;
    // the patch that the next store takes, once the store before the last has read it
    auto next_patch = [&]() {
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      __syncwarp();
      return patch0 + (stores & 1) * GG_PATCH_BYTES;
    };
    auto send_patch = [&](const CUtensorMap* map, uint8_t* patch, int c0, int c1, bool add) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        gg_store(map, c0, c1, smem_u32(patch), add);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
      ++stores;
    };
    for (int t = blockIdx.x; t < items && ok; t += gridDim.x) {
      const Item w = item_of(t);
      const CUtensorMap* map = w.seg == 0 ? &tmC0 : w.seg == 1 ? &tmC1 : &tmC2;
      const int row = w.g * a.out_rows + w.mt * 128 + q * 32, col0 = w.nt * 256;
      const bool rows_here = w.mt * 128 + q * 32 < a.M;  // (only a linear layer's last tile is shorter)
      const int per = a.out_f32 ? 32 : 64;               // columns of a patch
      if (w.beg >= w.end) {  // an expert without rows
        if (!a.add && rows_here) {
          for (int c = 0; c < 256 && col0 + c < a.N; c += per) {
            uint4* p = reinterpret_cast<uint4*>(next_patch());
#pragma unroll
            for (int i = 0; i < 8; ++i) p[lane * 8 + i] = make_uint4(0, 0, 0, 0);
            send_patch(map, reinterpret_cast<uint8_t*>(p), col0 + c, row, false);
          }
        }
        continue;
      }
      const int step = piece(w);
      for (int beg = w.beg; beg < w.end; beg += step, ++n) {
        const uint32_t buf = n & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->tmem_full[buf]), (n >> 1) & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t tb = tmem_base + ((uint32_t)(q * 32) << 16) + buf * 256;
        const bool add = a.add || beg > w.beg;
        if (beg > w.beg) {  // the piece before this one is in memory before this one is added to it
          if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
          __syncwarp();
        }
        if (rows_here) {
#pragma unroll 1
          for (int c = 0; c < 256 && col0 + c < a.N; c += per) {
            uint32_t v0[16], v1[16];
            tc_ld_issue(tb + c, v0);
            tc_ld_issue(tb + c + 16, v1);
            uint4* p = reinterpret_cast<uint4*>(next_patch());
            tc_ld_wait(v0, v1);
            auto put = [&](int i, uint4 v) { p[lane * 8 + (i ^ (lane & 7))] = v; };  // the 128-byte swizzle
            if (a.out_f32) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                put(i, make_uint4(v0[4 * i], v0[4 * i + 1], v0[4 * i + 2], v0[4 * i + 3]));
                put(4 + i, make_uint4(v1[4 * i], v1[4 * i + 1], v1[4 * i + 2], v1[4 * i + 3]));
              }
            } else {
              auto pack = [](uint32_t x, uint32_t y) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(x), __uint_as_float(y));
                return *reinterpret_cast<const uint32_t*>(&b);
              };
              auto put16 = [&](int i, const uint32_t (&v)[16]) {
                put(i, make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7])));
                put(i + 1, make_uint4(pack(v[8], v[9]), pack(v[10], v[11]), pack(v[12], v[13]), pack(v[14], v[15])));
              };
              put16(0, v0);
              put16(2, v1);
              tc_ld_issue(tb + c + 32, v0);
              tc_ld_issue(tb + c + 48, v1);
              tc_ld_wait(v0, v1);
              put16(4, v0);
              put16(6, v1);
            }
            send_patch(map, reinterpret_cast<uint8_t*>(p), col0 + c, row, add);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->tmem_empty[buf]));
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // shared memory is read, results are written
  }

  // ---- teardown: every role arrives here, also after a time-out ---------------------------------------
  tc_fence_before();
  __syncthreads();
  if (sh->abort_flag) {
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, B200MOE_STATUS_WAIT_TIMEOUT);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies and MMAs still in flight land before memory is released
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

// row-major matrix of bf16 or fp32 [rows, cols], boxes of `box_rows` rows x 128 bytes, 128-byte swizzle
bool gg_make_map(CUtensorMap* m, const void* base, bool f32, uint64_t rows, uint64_t cols, uint32_t box_rows) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return false;
  const uint64_t es = f32 ? 4 : 2;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {cols * es};
  cuuint32_t box[2] = {(cuuint32_t)(128 / es), box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
             strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool ROWS>
int gg_launch(const CUtensorMap (&tm)[6], const GgArgs& a, cudaStream_t st) {
  static bool attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return B200MOE_EDRIVER;
  if (!attr_set[dev]) {  // per-device attribute
    cudaFuncSetAttribute(gemm_grad_kernel<ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GG_SMEM_BYTES);
    attr_set[dev] = true;
  }
  const int64_t items = (int64_t)a.groups * a.segs * a.MT * a.NT;
  if (items >= (int64_t(1) << 31)) return B200MOE_ESHAPE;
  const int sms = moe_device_sm_count();
  return moe_launch_as(true, 1, gemm_grad_kernel<ROWS>, (unsigned)(items < sms ? items : sms), GG_THREADS, GG_SMEM_BYTES, st, tm[0],
                       tm[1], tm[2], tm[3], tm[4], tm[5], a);
}

}  // namespace

int moe_weight_grad_tc(const MoeWeightGradArgs& g, cudaStream_t st) {
  CUtensorMap tm[6];
  const int64_t acols = (int64_t)g.segs * g.M;
  if (!gg_make_map(&tm[0], g.a, false, (uint64_t)g.P, (uint64_t)acols, GG_BK)) return B200MOE_EDRIVER;
  if (!gg_make_map(&tm[1], g.b0, false, (uint64_t)g.P, (uint64_t)g.N, GG_BK)) return B200MOE_EDRIVER;
  if (!gg_make_map(&tm[2], g.b1 ? g.b1 : g.b0, false, (uint64_t)g.P, (uint64_t)g.N, GG_BK)) return B200MOE_EDRIVER;
  for (int i = 0; i < 3; ++i)
    if (!gg_make_map(&tm[3 + i], g.out[i < g.segs ? i : 0], g.out_f32, (uint64_t)g.groups * g.M, (uint64_t)g.N, 32)) return B200MOE_EDRIVER;
  GgArgs a{};
  a.offsets = g.offsets;
  a.P = (int)g.P;
  a.groups = g.groups, a.segs = g.segs;
  a.M = g.M, a.N = g.N;
  a.MT = (g.M + 127) / 128, a.NT = (g.N + 255) / 256;
  a.out_rows = g.M;
  a.chunk = g.out_f32 ? kGradChunk : 0;  // (what bf16 rounds away is larger than the sums' error)
  a.out_f32 = g.out_f32, a.add = g.add;
  a.status = g.status;
  return gg_launch<false>(tm, a, st);
}

int moe_row_product_tc(__nv_bfloat16* out, const __nv_bfloat16* a16, const __nv_bfloat16* b, int64_t rows, int K, int b_rows, int b_cycle,
                       int N, int32_t* status, cudaStream_t st) {
  CUtensorMap tm[6];
  if (!gg_make_map(&tm[0], a16, false, (uint64_t)rows, (uint64_t)K, 128)) return B200MOE_EDRIVER;
  if (!gg_make_map(&tm[1], b, false, (uint64_t)b_rows, (uint64_t)N, GG_BK)) return B200MOE_EDRIVER;
  if (!gg_make_map(&tm[3], out, false, (uint64_t)rows, (uint64_t)N, 32)) return B200MOE_EDRIVER;
  tm[2] = tm[1], tm[4] = tm[5] = tm[3];
  GgArgs a{};
  a.groups = a.segs = 1;
  a.M = (int)rows, a.N = N;
  a.MT = (int)((rows + 127) / 128), a.NT = (N + 255) / 256;
  a.K = K, a.kb_rows = b_cycle;
  a.status = status;
  return gg_launch<true>(tm, a, st);
}
