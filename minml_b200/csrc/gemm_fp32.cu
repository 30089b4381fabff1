/*
 * gemm_fp32.cu -- fp32 matrix products that keep fp32 accuracy at any K, on the TF32 tensor cores.
 *
 * Every element is split into hi, its upper 19 bits, which is what the tensor core reads of the fp32 tile as it lies in shared memory, and
 * lo = x - hi rounded to TF32, which warps write to a tile of their own; hi hi + hi lo + lo hi is accumulated.  Dropped are lo lo, at most
 * 2^-20 of the product and 2^-22 on average, and lo's rounding, 2^-21.  But the tensor core cuts its sums instead of rounding them, measured
 * 2e-8 of the sum for every 8 K indices and product, always toward zero: 3.7e-6 at K = 512 and 5.7e-5 at K = 8192, where an fp32 sum is off
 * by 4e-7 and 7e-7.  So an accumulator here takes one stage, 32 K indices (12 instructions, 2.3e-7), and the epilogue warps add it to sums that
 * they hold in registers, 64 columns a lane; four accumulators in tensor memory keep the tensor core ahead of them.
 * One CTA per SM, persistent over 128 x 128 tiles and, where there are few tiles, K ranges whose sums a second kernel adds up:
 *   warp 0 TMA, warp 1 multiplications, warps 2-9 sums and results, warps 10-13 split.
 * Shared-memory bandwidth bounds it (a stage is read and written by the copy, the split and three products).
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
		constexpr int OPERAND_BYTES = 128 * 128;
		constexpr int STAGE_BYTES = 2 * OPERAND_BYTES;
		constexpr int STAGES = 4, LO_STAGES = 2, BUFFERS = 4;
		constexpr int EPI_WARPS = 8, SPLIT_WARPS = 4;
		constexpr int THREADS = (2 + EPI_WARPS + SPLIT_WARPS) * 32;
		constexpr int BOX_BYTES = 32 * 128; // per epilogue warp: 32 x 32 results
		constexpr int SMEM_BYTES = (STAGES + LO_STAGES) * STAGE_BYTES + EPI_WARPS * BOX_BYTES + 1024;

		struct Params
		{
				int M, N, k_blocks;
				int a_mn, b_mn;
				int m_tiles, n_tiles, splits, blocks_per_split;
				float *d; // splits > 1: [splits, M, ldd] sums
				int ldd;
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

		__global__ void __launch_bounds__(THREADS, 1) kernel_gemm_fp32(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p)
		{
			extern __shared__ uint8_t smem_raw[];
			__shared__ Barriers bars;
			const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
			const uint32_t lo_base = smem_base + STAGES * STAGE_BYTES;
			const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
			const int tiles = p.m_tiles * p.n_tiles, units = tiles * p.splits;
			struct Unit
			{
					int m0, n0, kb0, kb1, split;
			};
			auto locate = [&](int unit) -> Unit
			{ // column tiles fastest within a K range
				Unit u;
				u.split = unit / tiles;
				const int rest = unit - u.split * tiles;
				u.m0 = rest / p.n_tiles * BM;
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
					mbar_init(smem_u32(&bars.split[s]), SPLIT_WARPS);
					mbar_init(smem_u32(&bars.empty[s]), 1);
				}
				for (int s = 0; s < LO_STAGES; s++)
					mbar_init(smem_u32(&bars.lo_empty[s]), 1);
				for (int b = 0; b < BUFFERS; b++)
				{
					mbar_init(smem_u32(&bars.tmem_full[b]), 1);
					mbar_init(smem_u32(&bars.tmem_empty[b]), EPI_WARPS);
				}
				bars.abort_flag = 0;
				fence_mbar_init();
			}
			if (warp == 1)
			{
				tmem_alloc(smem_u32(&bars.tmem_base), BUFFERS * BN);
				tmem_relinquish();
			}
			tcgen05_fence_before();
			__syncthreads();
			tcgen05_fence_after();
			const uint32_t tmem_base = bars.tmem_base;
			volatile int *abort_flag = &bars.abort_flag;
			let_next_grid_start();
			wait_for_previous_grid();

			if (warp == 0)
			{ /* ------------------------------------------------ operands */
				if (elect_one())
				{
					prefetch_tensormap(&map_a);
					prefetch_tensormap(&map_b);
					uint32_t it = 0;
					bool ok = true;
					for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x)
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
							const uint32_t a = smem_base + s * STAGE_BYTES, b = a + OPERAND_BYTES;
							if (p.a_mn)
							{
#pragma unroll
								for (int j = 0; j < 4; j++)
									tma_load_3d(a + j * (OPERAND_BYTES / 4), &map_a, full, u.m0 + j * 32, kb * BK, 0);
							}
							else
								tma_load_3d(a, &map_a, full, kb * BK, u.m0, 0);
							if (p.b_mn)
							{
#pragma unroll
								for (int j = 0; j < 4; j++)
									tma_load_3d(b + j * (OPERAND_BYTES / 4), &map_b, full, u.n0 + j * 32, kb * BK, 0);
							}
							else
								tma_load_3d(b, &map_b, full, kb * BK, u.n0, 0);
						}
					}
				}
				__syncwarp();
			}
			else if (warp == 1)
			{ /* ------------------------------------------- multiplications */
				if (elect_one())
				{
					const uint32_t idesc = make_idesc_tf32(BN) | (p.a_mn ? (1u << 15) : 0u) | (p.b_mn ? (1u << 16) : 0u);
					// per instruction (8 K indices), in 16-byte units: 32 bytes along K, or 8 K indices of 128 bytes
					const uint32_t step_a = p.a_mn ? 64 : 2, step_b = p.b_mn ? 64 : 2;
					auto describe = [](uint32_t addr, bool mn) -> uint64_t
					{
						return mn ? make_desc_mn_sw128(addr, OPERAND_BYTES / 4, true) : make_desc_k_sw128(addr);
					};
					uint32_t it = 0;
					bool ok = true;
					for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x)
					{
						const Unit u = locate(unit);
						for (int kb = u.kb0; kb < u.kb1; kb++, it++)
						{
							const int s = it % STAGES, b = it % BUFFERS;
							if (!mbar_wait(smem_u32(&bars.tmem_empty[b]), ((it / BUFFERS) & 1u) ^ 1u, abort_flag) || !mbar_wait(smem_u32(&bars.split[s]), (it / STAGES) & 1u, abort_flag))
							{
								ok = false;
								break;
							}
							tcgen05_fence_after();
							fence_proxy_async_smem(); // lo was written by plain stores of the split warps
							const uint32_t d = tmem_base + b * BN;
							const uint32_t hi = smem_base + s * STAGE_BYTES, lo = lo_base + (it % LO_STAGES) * STAGE_BYTES;
							const uint64_t hi_a = describe(hi, p.a_mn), hi_b = describe(hi + OPERAND_BYTES, p.b_mn);
							const uint64_t lo_a = describe(lo, p.a_mn), lo_b = describe(lo + OPERAND_BYTES, p.b_mn);
							// the small products first: their sum is cut at its own size
#pragma unroll
							for (int k = 0; k < 4; k++)
								mma_ss<2>(d, hi_a + step_a * k, lo_b + step_b * k, idesc, k > 0 ? 1u : 0u);
#pragma unroll
							for (int k = 0; k < 4; k++)
								mma_ss<2>(d, lo_a + step_a * k, hi_b + step_b * k, idesc, 1u);
							mma_commit(smem_u32(&bars.lo_empty[it % LO_STAGES]));
#pragma unroll
							for (int k = 0; k < 4; k++)
								mma_ss<2>(d, hi_a + step_a * k, hi_b + step_b * k, idesc, 1u);
							mma_commit(smem_u32(&bars.empty[s]));
							mma_commit(smem_u32(&bars.tmem_full[b]));
						}
					}
				}
				__syncwarp();
			}
			else if (warp >= 2 + EPI_WARPS)
			{ /* ------------------------------------------- split: lo of every element */
				const int t = threadIdx.x - (2 + EPI_WARPS) * 32;
				uint32_t it = 0;
				bool ok = true;
				for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x)
				{
					const Unit u = locate(unit);
					for (int kb = u.kb0; kb < u.kb1; kb++, it++)
					{
						const int s = it % STAGES;
						if (!mbar_wait(smem_u32(&bars.lo_empty[it % LO_STAGES]), ((it / LO_STAGES) & 1u) ^ 1u, abort_flag) || !mbar_wait(smem_u32(&bars.full[s]), (it / STAGES) & 1u, abort_flag))
						{
							ok = false;
							break;
						}
						const uint32_t hi = smem_base + s * STAGE_BYTES, lo = lo_base + (it % LO_STAGES) * STAGE_BYTES;
						constexpr int PER_THREAD = STAGE_BYTES / 16 / (SPLIT_WARPS * 32), GROUP = 8;
#pragma unroll 1
						for (int g = 0; g < PER_THREAD; g += GROUP)
						{ // elementwise, so whatever swizzle the copy wrote is kept
							uint4 x[GROUP];
#pragma unroll
							for (int i = 0; i < GROUP; i++)
								x[i] = ld_shared_v4(hi + (t + (g + i) * SPLIT_WARPS * 32) * 16);
#pragma unroll
							for (int i = 0; i < GROUP; i++)
								st_shared_v4(lo + (t + (g + i) * SPLIT_WARPS * 32) * 16, make_uint4(low_part(x[i].x), low_part(x[i].y), low_part(x[i].z), low_part(x[i].w)));
						}
						fence_proxy_async_smem();
						__syncwarp();
						if (lane == 0)
							mbar_arrive(smem_u32(&bars.split[s]));
					}
				}
			}
			else
			{ /* ------------------------------------------------------------ sums and results */
				const int q = warp % 4, half = (warp - 2) / 4;
				uint32_t it = 0;
				bool ok = true;
				for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x)
				{
					const Unit u = locate(unit);
					float v[BN / 2];
#pragma unroll
					for (int j = 0; j < BN / 2; j++)
						v[j] = 0.0f;
					for (int kb = u.kb0; kb < u.kb1; kb++, it++)
					{
						const int b = it % BUFFERS;
						if (!mbar_wait_warp(smem_u32(&bars.tmem_full[b]), (it / BUFFERS) & 1u, abort_flag, 20u))
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
							mbar_arrive(smem_u32(&bars.tmem_empty[b]));
#pragma unroll
						for (int j = 0; j < 32; j++)
						{
							v[j] += __uint_as_float(r0[j]);
							v[32 + j] += __uint_as_float(r1[j]);
						}
					}
					if (!ok)
						break;
					// a lane holds 64 columns of one row; through shared memory, so that a store instruction covers 128 bytes of one row
					const int row0 = u.m0 + q * 32, rows = min(32, p.M - row0);
					const uint32_t box = lo_base + LO_STAGES * STAGE_BYTES + (warp - 2) * BOX_BYTES;
#pragma unroll
					for (int c = 0; c < 2; c++)
					{
						const int n = u.n0 + half * (BN / 2) + c * 32 + lane;
#pragma unroll
						for (int k = 0; k < 8; k++)
							st_shared_v4(box + lane * 128 + ((k ^ (lane & 7)) * 16), make_uint4(__float_as_uint(v[c * 32 + 4 * k]), __float_as_uint(v[c * 32 + 4 * k + 1]),
									__float_as_uint(v[c * 32 + 4 * k + 2]), __float_as_uint(v[c * 32 + 4 * k + 3])));
						__syncwarp();
						if (n < p.N)
						{
							float *dst = p.d + (static_cast<long long>(u.split) * p.M + row0) * p.ldd + n;
#pragma unroll 8
							for (int r = 0; r < rows; r++, dst += p.ldd)
							{
								const float x = ld_shared_f32(box + r * 128 + (((lane / 4) ^ (r & 7)) * 16) + lane % 4 * 4);
								*dst = p.beta != 0.0f ? x + p.beta * *dst : x;
							}
						}
						__syncwarp();
					}
				}
			}

			tcgen05_fence_before();
			__syncthreads();
			if (bars.abort_flag != 0)
			{
				if (threadIdx.x == 0 && p.status != nullptr)
					atomicExch(p.status, 1);
				__nanosleep(1000000); // give copies that are still in flight time to land before the CTA retires
			}
			if (warp == 1)
			{
				tcgen05_fence_after();
				tmem_dealloc(tmem_base, BUFFERS * BN);
			}
		}

		/* Four destination elements a thread (pitch is a multiple of four). */
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_pack_rows(T *__restrict__ dst, int pitch, long long padded_rows, const T *__restrict__ src, long long rows, int columns, const GridWalk walk)
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

	/* As pair_splits (gemm_pair.cu), with this kernel's figures: a K block of a tile 0.75 us. */
	namespace
	{
		int float_splits(mlContext_t ctx, int M, int N, int K)
		{
			const int sms = get(ctx)->sm_count;
			const long long tiles = static_cast<long long>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
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
				const double time = static_cast<double>((tiles * s + sms - 1) / sms) * (blocks * 0.75 + 1.5) + (s == 1 ? 0.0 : 4.0 + partial_bytes / 5.0e6);
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
		static bool configured_on[MAX_DEVICES] = { false }; // the opt-in is a per-device attribute of the kernel
		static std::mutex mutex;
		Context *c = get(ctx);
		cudaStream_t stream = use_stream(ctx);
		if (c->device < 0 || c->device >= MAX_DEVICES)
			return false;
		{
			std::lock_guard<std::mutex> lock(mutex);
			if (!configured_on[c->device])
				configured_on[c->device] = check_cuda(ctx, cudaFuncSetAttribute(kernel_gemm_fp32, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES), "gemm_fp32: shared memory opt-in");
			if (!configured_on[c->device])
				return false;
		}
		// an operand stored [rows, K]: boxes of 128 rows x 128 bytes of K; stored [K, rows]: 32 K indices x 128 bytes of rows, whose swizzle moves
		// 32-byte pieces (tc.cuh)
		auto encode = [&](CUtensorMap *map, const FloatOperand &o, int rows) -> bool
		{
			const uint64_t dims[3] = { static_cast<uint64_t>(o.mn ? rows : K), static_cast<uint64_t>(o.mn ? K : rows), 1 };
			const uint64_t strides[2] = { static_cast<uint64_t>(o.ld) * 4, static_cast<uint64_t>(o.ld) * 4 * dims[1] };
			const uint32_t box[3] = { 32, o.mn ? 32u : 128u, 1 };
			return encode_tensor_map(ctx, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, o.data, dims, strides, box, o.mn ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B);
		};
		CUtensorMap map_a, map_b;
		if (!encode(&map_a, a, M) || !encode(&map_b, b, N))
			return false;
		Params p;
		std::memset(&p, 0, sizeof(p));
		const int splits = float_splits(ctx, M, N, K), k_blocks = (K + BK - 1) / BK;
		p.M = M;
		p.N = N;
		p.k_blocks = k_blocks;
		p.a_mn = a.mn;
		p.b_mn = b.mn;
		p.m_tiles = (M + BM - 1) / BM;
		p.n_tiles = (N + BN - 1) / BN;
		p.blocks_per_split = (k_blocks + splits - 1) / splits;
		p.splits = splits;
		p.d = splits > 1 ? partials : d;
		p.ldd = splits > 1 ? partial_pitch(N) : ldd;
		p.beta = splits > 1 ? 0.0f : beta;
		p.status = c->dev_status;
		const long long units = static_cast<long long>(p.m_tiles) * p.n_tiles * splits;
		if (units > 0x3FFFFFFF)
		{
			record_error(ctx, "gemm_fp32: %d x %d tiles are too many for one launch", p.m_tiles, p.n_tiles);
			return false;
		}
		const cudaError_t status = launch_overlapped(kernel_gemm_fp32, dim3(static_cast<unsigned>(std::min<long long>(units, c->sm_count))), dim3(THREADS), SMEM_BYTES, stream, map_a, map_b, p);
		MB200_COUNT_LAUNCH();
		c->kernels_with_waits = true;
		if (!check_cuda(ctx, status, "gemm_fp32 launch"))
			return false;
		return splits == 1 || finish_sums<float>(ctx, d, ldd, M, N, partials, p.ldd, splits, 1.0f, nullptr, nullptr, beta);
	}
} /* namespace mb200 */
