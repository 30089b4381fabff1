/*
 * gemm_fp32.cu -- fp32 matrix products that keep fp32 accuracy at any K, on the TF32 tensor cores.
 *
 * Every element is split into hi, its upper 19 bits, which is what the tensor core reads of an fp32 value, and lo = x - hi rounded to TF32;
 * hi hi + hi lo + lo hi is accumulated.  Dropped are lo lo, at most 2^-20 of the product and 2^-22 on average, and lo's rounding, 2^-21.  But the
 * tensor core cuts its sums instead of rounding them, measured 2e-8 of the sum for every 8 K indices and product, always toward zero:
 * 3.7e-6 at K = 512 and 5.7e-5 at K = 8192, where an fp32 sum is off by 4e-7 and 7e-7.  So an accumulator here takes one stage, 32 K indices
 * (12 instructions, 2.3e-7), and the epilogue warps add it to sums that they hold in registers, 64 columns a lane.
 * A cluster of two CTAs computes 256 x 128 tiles (cta_group::2), persistent over tiles and, where there are few, K ranges whose sums a second
 * kernel adds up.  Where the transposed product has fewer tiles, it is the one computed, and stored transposed.
 *   warp 0 TMA, warp 1 multiplications (of the even CTA), warps 4-11 sums and results, warps 12-19 split, two groups that take stages in turn.
 * Shared memory would bound it: with one CTA a tile and both terms of both operands there, a stage took 1400 cycles for 770 of
 * multiplications.  So A's terms go to tensor memory (a lane a row, 64 columns a stage; as a side effect it does not matter how A is stored),
 * each CTA holds and splits half of B, and of B's hi the tile that TMA wrote serves.  What bounded it next was the time from a tile's arrival
 * to its split, 700 cycles of one group of warps (two: 2504 -> 2115 us below).  The even CTA issues multiplications that read the lo of B which
 * the odd one's warps wrote, so a split stage is reported with a release at cluster scope, of shared memory alone: of all memory it takes 950
 * cycles more, or 1 200 to 1 400 of a warp that only passes the report on (2205 us -> 2376 below).  Now the tensor core is busy 84 % of the time at 1.44 GHz, the clock under the power limit (4096 x 4096 x 8192).
 * Measured, gated block forward and backward, 2000 x 4001 x 3001: 2085 - 2450 us by the clock (3191 with one CTA a tile), 8192 x 2048 x 8192: 11.0 -
 * 12.0 ms, 206 - 225 TFLOP/s.
 */
#include "common.cuh"
#include "tc.cuh"
#include "epilogue.cuh"
#include "operands.cuh"
#include "gemm_pair.cuh"
#include "gemm_fp32.cuh"

#include <algorithm>
#include <cstring>
#include <mutex>

namespace mb200
{
	namespace
	{
		using namespace tc;
		using namespace epi;

		constexpr int BM = 128, BN = 128, BK = 32;
		constexpr int A_BYTES = BM * BK * 4, B_BYTES = BN / 2 * BK * 4; // of a CTA
		constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
		constexpr int STAGES = 5, LO_STAGES = 4, BUFFERS = 2;
		constexpr int A_COLUMNS = 2 * BK; // of tensor memory: hi and lo of a stage of A, a row a lane
		constexpr int TMEM_COLUMNS = 512;
		static_assert(BUFFERS * BN + LO_STAGES * A_COLUMNS <= TMEM_COLUMNS, "tensor memory");
		constexpr int EPI_FIRST = 4, EPI_WARPS = 8, SPLIT_FIRST = EPI_FIRST + EPI_WARPS, SPLIT_WARPS = 4, SPLIT_GROUPS = 2; // groups take stages in turn
		constexpr int THREADS = (SPLIT_FIRST + SPLIT_WARPS * SPLIT_GROUPS) * 32;
		// warps 0-3, the epilogue's and the split's; launched with 96 registers a thread
		constexpr int REGISTERS_FEW = 40, REGISTERS_EPILOGUE = 144, REGISTERS_SPLIT = 72;
		static_assert(128 * REGISTERS_FEW + 256 * REGISTERS_EPILOGUE + 256 * REGISTERS_SPLIT <= THREADS * 96, "registers of the block at launch");
		constexpr int BOX_MN_BYTES = BK * 128; // 32 rows of an operand that is stored [K, rows]
		constexpr int BOX_BYTES = 32 * 128; // 32 x 32 results, two an epilogue warp
		constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + LO_STAGES * B_BYTES + EPI_WARPS * 2 * BOX_BYTES + 1024;

		struct Params
		{
				int M, N, k_blocks;
				int a_mn, b_mn;
				int m_tiles, n_tiles, splits, blocks_per_split;
				float *d; // splits > 1: sums of each K range, split_stride elements apart
				int ldd;
				long long split_stride;
				int transposed; // d [N, ldd] takes the transpose
				int by_copies; // d is stored through map_d
				float beta;
				int *status;
		};
		struct Barriers
		{
				uint64_t full[STAGES], split[STAGES], empty[STAGES];
				uint64_t lo_empty[LO_STAGES];
				uint64_t tmem_full[BUFFERS], tmem_empty[BUFFERS];
				uint32_t tmem_base;
				int abort_flag;
		};
		/* What the upper 19 bits of x leave, rounded to TF32 (either way, so that the cut of the tensor core has nothing to cut). */
		__device__ __forceinline__ uint32_t low_part(uint32_t x)
		{
			const float lo = __uint_as_float(x) - __uint_as_float(x & 0xFFFFE000u);
			return (__float_as_uint(lo) + 0x1000u) & 0xFFFFE000u;
		}

		__global__ void __launch_bounds__(THREADS, 1) kernel_gemm_fp32(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
				const __grid_constant__ CUtensorMap map_d, const Params p)
		{
			extern __shared__ uint8_t smem_raw[];
			__shared__ Barriers bars;
			const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
			const uint32_t lo_base = smem_base + STAGES * STAGE_BYTES;
			const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
			const uint32_t rank = cluster_ctarank();
			const bool leader = rank == 0;
			const int tiles = p.m_tiles * p.n_tiles, units = tiles * p.splits, first_unit = blockIdx.x / 2, unit_step = gridDim.x / 2;
			struct Unit
			{
					int m0, n0, kb0, kb1, split;
			};
			auto locate = [&](int unit) -> Unit
			{ // column tiles fastest within a K range
				Unit u;
				u.split = unit / tiles;
				const int rest = unit - u.split * tiles;
				u.m0 = (rest / p.n_tiles * 2 + static_cast<int>(rank)) * BM;
				u.n0 = rest % p.n_tiles * BN;
				u.kb0 = u.split * p.blocks_per_split;
				u.kb1 = min(p.k_blocks, u.kb0 + p.blocks_per_split);
				return u;
			};

			if (threadIdx.x == 0)
			{
				for (int s = 0; s < STAGES; s++)
				{
					mbar_init(smem_u32(&bars.full[s]), 1);
					mbar_init(smem_u32(&bars.split[s]), 2 * SPLIT_WARPS);
					mbar_init(smem_u32(&bars.empty[s]), 1);
				}
				for (int s = 0; s < LO_STAGES; s++)
					mbar_init(smem_u32(&bars.lo_empty[s]), 1);
				for (int b = 0; b < BUFFERS; b++)
				{
					mbar_init(smem_u32(&bars.tmem_full[b]), 1);
					mbar_init(smem_u32(&bars.tmem_empty[b]), 2 * EPI_WARPS);
				}
				bars.abort_flag = 0;
				fence_mbar_init();
			}
			if (warp == 1)
			{
				asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&bars.tmem_base)), "r"(TMEM_COLUMNS) : "memory");
				asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
			}
			tcgen05_fence_before();
			cluster_sync(); // the peer's barriers exist before anything signals them
			tcgen05_fence_after();
			const uint32_t tmem_base = bars.tmem_base;
			volatile int *abort_flag = &bars.abort_flag;
			let_next_grid_start();
			wait_for_previous_grid();

			if (warp == 0)
			{ /* ------------------------------------------------ operands */
				asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(REGISTERS_FEW));
				if (elect_one())
				{
					prefetch_tensormap(&map_a);
					prefetch_tensormap(&map_b);
					uint32_t it = 0;
					bool ok = true;
					for (int unit = first_unit; unit < units && ok; unit += unit_step)
					{
						const Unit u = locate(unit);
						for (int kb = u.kb0; kb < u.kb1; kb++, it++)
						{
							const int s = it % STAGES;
							if (!mbar_wait(smem_u32(&bars.empty[s]), ((it / STAGES) & 1u) ^ 1u, abort_flag))
							{
								ok = false;
								break;
							}
							const uint32_t full = smem_u32(&bars.full[s]);
							mbar_arrive_expect_tx(full, STAGE_BYTES);
							const uint32_t a = smem_base + s * STAGE_BYTES, b = a + A_BYTES;
							const int n0 = u.n0 + static_cast<int>(rank) * (BN / 2); // this CTA's half of the columns
							if (p.a_mn)
							{
#pragma unroll
								for (int j = 0; j < 4; j++)
									tma_load_3d(a + j * BOX_MN_BYTES, &map_a, full, u.m0 + j * 32, kb * BK, 0);
							}
							else
								tma_load_3d(a, &map_a, full, kb * BK, u.m0, 0);
							if (p.b_mn)
							{
#pragma unroll
								for (int j = 0; j < 2; j++)
									tma_load_3d(b + j * BOX_MN_BYTES, &map_b, full, n0 + j * 32, kb * BK, 0);
							}
							else
								tma_load_3d(b, &map_b, full, kb * BK, n0, 0);
						}
					}
				}
				__syncwarp();
			}
			else if (warp == 1)
			{ /* ------------------------------------------- multiplications */
				asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(REGISTERS_FEW));
				if (leader && elect_one())
				{
					const uint32_t idesc = make_idesc_tf32_pair(BN) | (p.b_mn ? (1u << 16) : 0u);
					// per instruction (8 K indices): 8 columns of A; of B, in 16-byte units, 32 bytes along K, or 8 K indices of 128 bytes
					const uint32_t step_b = p.b_mn ? 64 : 2;
					auto describe = [&](uint32_t addr) -> uint64_t
					{
						return p.b_mn ? make_desc_mn_sw128(addr, BOX_MN_BYTES, true) : make_desc_k_sw128(addr);
					};
					uint32_t it = 0;
					bool ok = true;
					for (int unit = first_unit; unit < units && ok; unit += unit_step)
					{
						const Unit u = locate(unit);
						for (int kb = u.kb0; kb < u.kb1; kb++, it++)
						{
							const int s = it % STAGES, b = it % BUFFERS;
							if (!mbar_wait_cluster(smem_u32(&bars.tmem_empty[b]), ((it / BUFFERS) & 1u) ^ 1u, abort_flag)
									|| !mbar_wait_cluster(smem_u32(&bars.split[s]), (it / STAGES) & 1u, abort_flag))
							{
								ok = false;
								break;
							}
							tcgen05_fence_after();
							fence_proxy_async_smem(); // lo was written by plain stores of the split warps
							const uint32_t d = tmem_base + b * BN;
							const uint32_t hi_a = tmem_base + BUFFERS * BN + (it % LO_STAGES) * A_COLUMNS, lo_a = hi_a + BK;
							const uint64_t hi_b = describe(smem_base + s * STAGE_BYTES + A_BYTES), lo_b = describe(lo_base + (it % LO_STAGES) * B_BYTES);
							// the small products first: their sum is cut at its own size
#pragma unroll
							for (int k = 0; k < 4; k++)
								mma_ts_tf32_pair(d, hi_a + 8 * k, lo_b + step_b * k, idesc, k > 0 ? 1u : 0u);
#pragma unroll
							for (int k = 0; k < 4; k++)
								mma_ts_tf32_pair(d, lo_a + 8 * k, hi_b + step_b * k, idesc, 1u);
#pragma unroll
							for (int k = 0; k < 4; k++)
								mma_ts_tf32_pair(d, hi_a + 8 * k, hi_b + step_b * k, idesc, 1u);
							mma_commit_pair(smem_u32(&bars.lo_empty[it % LO_STAGES]));
							mma_commit_pair(smem_u32(&bars.empty[s]));
							mma_commit_pair(smem_u32(&bars.tmem_full[b]));
						}
					}
				}
				__syncwarp();
			}
			else if (warp < EPI_FIRST)
				asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(REGISTERS_FEW));
			else if (warp >= SPLIT_FIRST)
			{ /* ------------------------------------------- split: A to tensor memory, lo of B to shared memory */
				asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(REGISTERS_SPLIT));
				const int t = threadIdx.x % (SPLIT_WARPS * 32), q = warp % 4;
				const uint32_t group = (warp - SPLIT_FIRST) / SPLIT_WARPS;
				uint32_t it = 0;
				bool ok = true;
				for (int unit = first_unit; unit < units && ok; unit += unit_step)
				{
					const Unit u = locate(unit);
					for (int kb = u.kb0; kb < u.kb1; kb++, it++)
					{
						const int s = it % STAGES;
						if (it % SPLIT_GROUPS != group)
							continue;
						if (!mbar_wait_all_lanes(smem_u32(&bars.lo_empty[it % LO_STAGES]), ((it / LO_STAGES) & 1u) ^ 1u, abort_flag)
								|| !mbar_wait_all_lanes(smem_u32(&bars.full[s]), (it / STAGES) & 1u, abort_flag))
						{
							ok = false;
							break;
						}
						tcgen05_fence_after();
						const uint32_t a = smem_base + s * STAGE_BYTES, hi = a + A_BYTES, lo = lo_base + (it % LO_STAGES) * B_BYTES;
						const uint32_t to = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + BUFFERS * BN + (it % LO_STAGES) * A_COLUMNS;
						// a lane's row of A, 16 K indices at a time
#pragma unroll
						for (int c = 0; c < BK; c += 16)
						{
							uint32_t x[16], low[16];
							if (p.a_mn)
							{ // [block of 32 rows][K index][row]
#pragma unroll
								for (int k = 0; k < 16; k++)
									x[k] = __float_as_uint(ld_shared_f32(a + q * BOX_MN_BYTES + (c + k) * 128 + lane * 4));
							}
							else
							{ // [row][K index], 16-byte pieces swizzled
#pragma unroll
								for (int k = 0; k < 4; k++)
								{
									const uint4 v = ld_shared_v4(a + (q * 32 + lane) * 128 + (((c / 4 + k) ^ (lane & 7)) * 16));
									x[4 * k] = v.x;
									x[4 * k + 1] = v.y;
									x[4 * k + 2] = v.z;
									x[4 * k + 3] = v.w;
								}
							}
#pragma unroll
							for (int k = 0; k < 16; k++)
							{
								low[k] = low_part(x[k]);
								x[k] &= 0xFFFFE000u;
							}
							tmem_st_32x16(to + c, x);
							tmem_st_32x16(to + BK + c, low);
						}
						constexpr int PER_THREAD = B_BYTES / 16 / (SPLIT_WARPS * 32);
						uint4 x[PER_THREAD]; // of B, elementwise, so whatever swizzle the copy wrote is kept
#pragma unroll
						for (int i = 0; i < PER_THREAD; i++)
							x[i] = ld_shared_v4(hi + (t + i * SPLIT_WARPS * 32) * 16);
#pragma unroll
						for (int i = 0; i < PER_THREAD; i++)
							st_shared_v4(lo + (t + i * SPLIT_WARPS * 32) * 16, make_uint4(low_part(x[i].x), low_part(x[i].y), low_part(x[i].z), low_part(x[i].w)));
						tmem_wait_st();
						tcgen05_fence_before();
						fence_proxy_async_smem();
						__syncwarp();
						if (lane == 0)
							publish_to_leader(smem_u32(&bars.split[s]));
					}
				}
			}
			else
			{ /* ------------------------------------------------------------ sums and results */
				asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(REGISTERS_EPILOGUE));
				const int q = warp % 4, half = (warp - EPI_FIRST) / 4;
				const uint32_t boxes = lo_base + LO_STAGES * B_BYTES + (warp - EPI_FIRST) * 2 * BOX_BYTES;
				uint32_t it = 0;
				bool ok = true;
				for (int unit = first_unit; unit < units && ok; unit += unit_step)
				{
					const Unit u = locate(unit);
					float v[BN / 2];
#pragma unroll
					for (int j = 0; j < BN / 2; j++)
						v[j] = 0.0f;
					for (int kb = u.kb0; kb < u.kb1; kb++, it++)
					{
						const int b = it % BUFFERS;
						if (!mbar_wait_all_lanes(smem_u32(&bars.tmem_full[b]), (it / BUFFERS) & 1u, abort_flag))
						{
							ok = false;
							break;
						}
						tcgen05_fence_after();
						const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * BN + half * (BN / 2);
						uint32_t r0[32], r1[32];
						tmem_ld_32x32(taddr, r0);
						tmem_ld_32x32(taddr + 32, r1);
						tmem_wait_ld();
						tcgen05_fence_before();
						__syncwarp();
						if (lane == 0)
							arrive_at_leader(smem_u32(&bars.tmem_empty[b]));
#pragma unroll
						for (int j = 0; j < 32; j++)
						{
							v[j] += __uint_as_float(r0[j]);
							v[32 + j] += __uint_as_float(r1[j]);
						}
					}
					if (!ok)
						break;
					// a lane holds 64 columns of one row: to boxes of 32 x 32 of the result, which the copy engine stores while the next tile is summed
					// up, or, where it cannot (beta, alignment), the warp stores 128 bytes of a row at a time
					const int result_rows = p.transposed ? p.N : p.M, result_columns = p.transposed ? p.M : p.N;
					if (lane == 0)
						bulk_wait_group_read<0>(); // of the last tile's boxes
					__syncwarp();
#pragma unroll
					for (int c = 0; c < 2; c++)
					{
						const uint32_t box = boxes + c * BOX_BYTES;
						const int along_m = u.m0 + q * 32, along_n = u.n0 + half * (BN / 2) + c * 32;
						const int row0 = p.transposed ? along_n : along_m, column0 = p.transposed ? along_m : along_n;
						if (p.transposed)
						{
#pragma unroll
							for (int j = 0; j < 32; j++)
								st_shared_f32(box + j * 128 + (((lane / 4) ^ (j & 7)) * 16) + lane % 4 * 4, v[c * 32 + j]);
						}
						else
						{
#pragma unroll
							for (int k = 0; k < 8; k++)
								st_shared_v4(box + lane * 128 + ((k ^ (lane & 7)) * 16), make_uint4(__float_as_uint(v[c * 32 + 4 * k]), __float_as_uint(v[c * 32 + 4 * k + 1]),
										__float_as_uint(v[c * 32 + 4 * k + 2]), __float_as_uint(v[c * 32 + 4 * k + 3])));
						}
						if (p.by_copies)
						{
							fence_proxy_async_smem();
							__syncwarp();
							if (lane == 0 && row0 < result_rows && column0 < result_columns)
								tma_store_3d(&map_d, box, column0, row0, u.split);
							continue;
						}
						__syncwarp();
						const int rows = min(32, result_rows - row0), column = column0 + lane;
						if (column < result_columns)
						{
							float *dst = p.d + u.split * p.split_stride + static_cast<long long>(row0) * p.ldd + column;
#pragma unroll 8
							for (int r = 0; r < rows; r++, dst += p.ldd)
							{
								const float x = ld_shared_f32(box + r * 128 + (((lane / 4) ^ (r & 7)) * 16) + lane % 4 * 4);
								*dst = p.beta != 0.0f ? x + p.beta * *dst : x;
							}
						}
					}
					if (lane == 0)
						bulk_commit_group();
				}
				if (lane == 0)
					bulk_wait_group_read<0>(); // shared memory stays until the last store has read it
				__syncwarp();
			}

			tcgen05_fence_before();
			__syncthreads();
			if (bars.abort_flag != 0)
			{
				if (threadIdx.x == 0 && p.status != nullptr)
					atomicExch(p.status, 1);
				__nanosleep(1000000); // give copies that are still in flight time to land before the CTA retires
			}
			cluster_sync(); // neither CTA's shared or tensor memory goes while the other may still use it
			if (warp == 1)
			{
				tcgen05_fence_after();
				asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem_base), "r"(TMEM_COLUMNS) : "memory");
			}
		}

		/* Four destination elements a thread (pitch is a multiple of four). */
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_pack_rows(T *dst, int pitch, long long padded_rows, const T *src, long long rows, int columns, const GridWalk walk)
		{
			struct alignas(4 * sizeof(T)) Four
			{
					T v[4];
			};
			let_next_grid_start();
			wait_for_previous_grid();
			const long long stride = static_cast<long long>(gridDim.x) * 256;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < walk.total; i += stride)
			{
				long long r;
				int c;
				walk.place(i, r, c);
				c *= 4;
				long long block = 0, inside = r;
				for (; inside >= padded_rows; inside -= padded_rows) // at most two blocks
					block++;
				const T *from = src + (block * rows + inside) * columns + c;
				Four out;
#pragma unroll
				for (int k = 0; k < 4; k++)
					out.v[k] = inside < rows && c + k < columns ? from[k] : from_float<T>(0.0f);
				*reinterpret_cast<Four*>(dst + r * pitch + c) = out;
			}
		}
	}

	template<typename T>
	bool pack_rows(mlContext_t ctx, T *dst, int pitch, long long padded_rows, const T *src, long long rows, int columns, int blocks)
	{
		const long long threads = padded_rows * blocks * (pitch / 4);
		const int grid = static_cast<int>(std::max<long long>(1, std::min<long long>((threads + 255) / 256, static_cast<long long>(get(ctx)->sm_count) * 16)));
		const cudaError_t status = launch_overlapped(kernel_pack_rows<T>, dim3(grid), dim3(256), 0, use_stream(ctx), dst, pitch, padded_rows, src, rows, columns,
				GridWalk(padded_rows * blocks, pitch / 4));
		MB200_COUNT_LAUNCH();
		return check_cuda(ctx, status, "pack_rows");
	}
	template bool pack_rows<__half>(mlContext_t, __half*, int, long long, const __half*, long long, int, int);
	template bool pack_rows<float>(mlContext_t, float*, int, long long, const float*, long long, int, int);

	/* As pair_splits (gemm_pair.cu), with this kernel's figures: a K block of a tile 0.6 us, the rest of a tile 2, the second kernel 2 and its traffic. */
	namespace
	{
		/* How many clusters the device holds at once; 0 when they cannot be placed.  Also opts the kernel in to its shared memory; both once per device. */
		int resident_clusters(mlContext_t ctx)
		{
			static int known[MAX_DEVICES] = { 0 }; // 0: not asked yet, -1: none
			static std::mutex mutex;
			std::lock_guard<std::mutex> lock(mutex);
			const int device = get(ctx)->device;
			if (device < 0 || device >= MAX_DEVICES)
				return 0;
			if (known[device] == 0)
			{
				use_stream(ctx);
				int n = 0;
				cudaLaunchConfig_t config = { };
				cudaLaunchAttribute attribute = { };
				attribute.id = cudaLaunchAttributeClusterDimension;
				attribute.val.clusterDim.x = 2;
				attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
				config.gridDim = dim3(2 * (get(ctx)->sm_count / 2));
				config.blockDim = dim3(THREADS);
				config.dynamicSmemBytes = SMEM_BYTES;
				config.attrs = &attribute;
				config.numAttrs = 1;
				if (cudaFuncSetAttribute(kernel_gemm_fp32, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess
						|| cudaOccupancyMaxActiveClusters(&n, kernel_gemm_fp32, &config) != cudaSuccess || n <= 0)
				{
					cudaGetLastError();
					n = -1;
				}
				known[device] = n;
			}
			return std::max(0, known[device]);
		}
		/* Tiles of 256 x 128; the product's transpose, where it has fewer (300 rows are 384 as columns, 512 as rows). */
		long long tiles_of(int M, int N)
		{
			return static_cast<long long>((M + 2 * BM - 1) / (2 * BM)) * ((N + BN - 1) / BN);
		}
		bool takes_transpose(int M, int N)
		{
			return tiles_of(N, M) < tiles_of(M, N);
		}
		int float_splits(mlContext_t ctx, int M, int N, int K)
		{
			const int clusters = std::max(1, resident_clusters(ctx));
			const long long tiles = std::min(tiles_of(M, N), tiles_of(N, M));
			const int k_blocks = (K + BK - 1) / BK;
			int best = 1;
			double best_time = 0.0;
			for (int s = 1; s <= 64 && tiles > 0 && (s == 1 || k_blocks / s >= 4); s++)
			{
				const int blocks = (k_blocks + s - 1) / s;
				if ((k_blocks + blocks - 1) / blocks != s)
					continue;
				const double partial_bytes = s == 1 ? 0.0 : 8.0 * s * M * N;
				if (partial_bytes > 2.0 * (size_t(256) << 20))
					break;
				const double time = static_cast<double>((tiles * s + clusters - 1) / clusters) * (blocks * 0.6 + 2.0) + (s == 1 ? 0.0 : 2.0 + partial_bytes / 5.0e6);
				if (s == 1 || time < best_time)
				{
					best = s;
					best_time = time;
				}
			}
			return best;
		}
		int partial_pitch(int N)
		{
			return (N + 3) / 4 * 4;
		}
	}
	size_t float_partial_elements(mlContext_t ctx, int M, int N, int K)
	{
		const int splits = float_splits(ctx, M, N, K);
		return splits == 1 ? 0 : static_cast<size_t>(splits) * M * partial_pitch(N);
	}
	bool float_product(mlContext_t ctx, int M, int N, int K, const FloatOperand &a, const FloatOperand &b, float *d, int ldd, float beta, float *partials)
	{
		Context *c = get(ctx);
		const int resident = resident_clusters(ctx);
		if (resident == 0)
		{
			record_error(ctx, "gemm_fp32: a cluster of two CTAs with %d bytes of shared memory each cannot be placed on this device", SMEM_BYTES);
			return false;
		}
		// an operand stored [rows, K]: boxes of 128 rows x 128 bytes of K; stored [K, rows]: 32 K indices x 128 bytes of rows, whose swizzle moves
		// 32-byte pieces (tc.cuh)
		auto encode = [&](CUtensorMap *map, const FloatOperand &o, int rows, uint32_t box_rows, CUtensorMapSwizzle swizzle_mn) -> bool
		{
			const uint64_t dims[3] = { static_cast<uint64_t>(o.mn ? rows : K), static_cast<uint64_t>(o.mn ? K : rows), 1 };
			const uint64_t strides[2] = { static_cast<uint64_t>(o.ld) * 4, static_cast<uint64_t>(o.ld) * 4 * dims[1] };
			const uint32_t box[3] = { 32, o.mn ? 32u : box_rows, 1 };
			return encode_tensor_map(ctx, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, o.data, dims, strides, box, o.mn ? swizzle_mn : CU_TENSOR_MAP_SWIZZLE_128B);
		};
		const bool transposed = takes_transpose(M, N);
		const FloatOperand &first = transposed ? b : a, &second = transposed ? a : b;
		const int rows = transposed ? N : M, columns = transposed ? M : N; // of what the kernel multiplies
		CUtensorMap map_a, map_b;
		if (!encode(&map_a, first, rows, BM, CU_TENSOR_MAP_SWIZZLE_NONE) || !encode(&map_b, second, columns, BN / 2, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B))
			return false;
		Params p;
		std::memset(&p, 0, sizeof(p));
		const int splits = float_splits(ctx, M, N, K), k_blocks = (K + BK - 1) / BK;
		p.M = rows;
		p.N = columns;
		p.transposed = transposed;
		p.k_blocks = k_blocks;
		p.a_mn = first.mn;
		p.b_mn = second.mn;
		p.m_tiles = (rows + 2 * BM - 1) / (2 * BM);
		p.n_tiles = (columns + BN - 1) / BN;
		p.blocks_per_split = (k_blocks + splits - 1) / splits;
		p.splits = splits;
		p.d = splits > 1 ? partials : d;
		p.ldd = splits > 1 ? partial_pitch(N) : ldd;
		p.split_stride = static_cast<long long>(M) * p.ldd;
		p.beta = splits > 1 ? 0.0f : beta;
		p.status = c->dev_status;
		CUtensorMap map_d = map_a; // unused unless by_copies
		p.by_copies = p.beta == 0.0f && p.ldd % 4 == 0 && aligned_to(p.d, 16);
		if (p.by_copies)
		{
			const uint64_t dims[3] = { static_cast<uint64_t>(N), static_cast<uint64_t>(M), static_cast<uint64_t>(splits) };
			const uint64_t strides[2] = { static_cast<uint64_t>(p.ldd) * 4, static_cast<uint64_t>(p.split_stride) * 4 };
			const uint32_t box[3] = { 32, 32, 1 };
			if (!encode_tensor_map(ctx, &map_d, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, p.d, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
				return false;
		}
		const long long units = static_cast<long long>(p.m_tiles) * p.n_tiles * splits;
		if (units > 0x3FFFFFFF)
		{
			record_error(ctx, "gemm_fp32: %d x %d tiles are too many for one launch", p.m_tiles, p.n_tiles);
			return false;
		}
		cudaLaunchConfig_t config = { };
		cudaLaunchAttribute attributes[2] = { };
		attributes[0].id = cudaLaunchAttributeClusterDimension;
		attributes[0].val.clusterDim.x = 2;
		attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
		attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
		attributes[1].val.programmaticStreamSerializationAllowed = 1;
		config.gridDim = dim3(2 * static_cast<unsigned>(std::min<long long>(units, resident)));
		config.blockDim = dim3(THREADS);
		config.dynamicSmemBytes = SMEM_BYTES;
		config.stream = use_stream(ctx);
		config.attrs = attributes;
		config.numAttrs = 2;
		const cudaError_t status = cudaLaunchKernelEx(&config, kernel_gemm_fp32, map_a, map_b, map_d, p);
		MB200_COUNT_LAUNCH();
		if (!check_cuda(ctx, status, "gemm_fp32 launch"))
			return false;
		return splits == 1 || finish_sums<float>(ctx, d, ldd, M, N, partials, p.ldd, splits, 1.0f, nullptr, nullptr, beta);
	}
} /* namespace mb200 */
