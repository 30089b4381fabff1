/*
 * few_rows.cu -- products of a few rows x [T, K] with a weight matrix W [N, K], in fp32 arithmetic: bound by reading W once.
 *
 * An fp32 weight is 4 bytes for T multiply-adds, which the fp32 units keep up with (1.6 T weights a second x 16 = 26 of their 37 T), so nothing
 * has to be split into TF32 terms for the tensor cores; and lanes read consecutive elements of a row wherever it starts (by fours or twos where
 * the row length and the addresses allow), so rows of any length are read in place, where the tensor-core paths first copy them to padded rows
 * at three times the traffic.
 * A warp takes 4 weight rows, 8 for more than two tokens (GATED: half of them gate rows, half the matching up rows) and a stretch of K.  x comes
 * from L1 (or, a long one, L2) once for all the warp's rows: with 4 rows at 8 tokens it was twice the weights' traffic, 254 us to 134 below.  A
 * block is warps_n x warps_k = 8 warps: as many share a row's K as it takes for 8 blocks an SM, so that the last round of blocks is a small part
 * of the whole.  Sums: one fp32 chain a lane, halved over the lanes (each step sends half of the sums away, so 32 of them cost 31 shuffles), then
 * over the warps in their order.
 * Measured, fp32, embed 4096, hidden 11008, both products: 1 token 82 us (541 MB at 6.6 TB/s), 8 tokens 134, 16 tokens 211 (bound by the loads of x
 * and the latency of 8 warps an SM); embed 4097, hidden 11009, read singly: 95, 145, 299.  fp16, embed 4097, hidden 11009: 71 and 135 (1 and 8).
 * Logits' statistics, embed 2048, V = 50021: 65, 92, 161.
 */
#include "common.cuh"
#include "gate.cuh"
#include "operands.cuh"
#include "few_rows.cuh"

namespace mb200
{
	namespace
	{
		constexpr int WARPS = 8, MIN_STRETCH = 256; // of K, for a warp
		enum Kind
		{
			GATED,
			PRODUCT,
			STATISTICS
		};
		template<typename T>
		struct Params
		{
				int tokens, K, N; // N: columns of the result (GATED: of h)
				int warps_k;
				const T *x, *w;
				T *out;
				float *au;
				int gate;
				float beta;
				const int *targets;
				float2 *parts;
				float *target_logit;
		};
		/* Weight rows of a warp, for so many tokens. */
		constexpr int rows_of_warp(int tokens)
		{
			return tokens <= 2 ? 4 : 8;
		}
		template<typename T, int VEC>
		struct alignas(sizeof(T) * VEC) Piece
		{
				T v[VEC];
		};
		/* Weights are read once and leave L1 to x. */
		template<typename T, int VEC>
		__device__ __forceinline__ Piece<T, VEC> load_weights(const T *src)
		{
			constexpr int BYTES = sizeof(T) * VEC;
			Piece<T, VEC> p;
			if constexpr (BYTES == 16)
			{
				uint4 v;
				asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(src));
				memcpy(&p, &v, BYTES);
			}
			else if constexpr (BYTES == 8)
			{
				uint2 v;
				asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(src));
				memcpy(&p, &v, BYTES);
			}
			else if constexpr (BYTES == 4)
			{
				uint32_t v;
				asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(v) : "l"(src));
				memcpy(&p, &v, BYTES);
			}
			else
			{
				uint16_t v;
				asm volatile("ld.global.L1::no_allocate.b16 %0, [%1];" : "=h"(v) : "l"(src));
				memcpy(&p, &v, BYTES);
			}
			return p;
		}
		__device__ float gate_by_code(int gate, float g)
		{
			switch (gate)
			{
				case MB200_GATE_SIGMOID:
					return gate_value<MB200_GATE_SIGMOID, false>(g);
				case MB200_GATE_RELU:
					return gate_value<MB200_GATE_RELU, false>(g);
				case MB200_GATE_GELU:
					return gate_value<MB200_GATE_GELU, false>(g);
				default:
					return gate_value<MB200_GATE_SILU, false>(g);
			}
		}

		/* Lane l ends with the warp's sums of values [l COUNT / 32, (l + 1) COUNT / 32), or, with fewer than 32, 32 / COUNT lanes with the same one. */
		template<int LEFT, int DISTANCE, int COUNT>
		__device__ __forceinline__ void sum_over_lanes(float (&v)[COUNT], int lane)
		{
			if constexpr (DISTANCE >= 1)
			{
				constexpr int HALF = LEFT / 2;
				if constexpr (HALF >= 1)
				{
					const bool upper = lane & DISTANCE;
#pragma unroll
					for (int i = 0; i < HALF; i++)
					{
						const float away = upper ? v[i] : v[i + HALF], keep = upper ? v[i + HALF] : v[i];
						v[i] = keep + __shfl_xor_sync(0xffffffffu, away, DISTANCE);
					}
				}
				else
					v[0] += __shfl_xor_sync(0xffffffffu, v[0], DISTANCE);
				sum_over_lanes<HALF >= 1 ? HALF : 1, DISTANCE / 2>(v, lane);
			}
		}
		template<typename T, int VEC, int KIND, int TOKENS>
		__global__ void __launch_bounds__(WARPS * 32, TOKENS > 8 ? 1 : 2) kernel_few_rows(const Params<T> p)
		{
			constexpr int ROWS = rows_of_warp(TOKENS), STEP = 32 * VEC, UNROLL = (VEC == 4 ? 8 : 16) / ROWS, SUMS = ROWS * TOKENS, COLUMNS = KIND == GATED ? ROWS / 2 : ROWS; // of a warp
			static_assert((SUMS & (SUMS - 1)) == 0, "halved down to one a lane");
			__shared__ float sums[WARPS][SUMS];
			const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
			const int warps_n = WARPS / p.warps_k, columns = warps_n * COLUMNS; // of the block
			const int n0 = blockIdx.x * columns + warp / p.warps_k * COLUMNS;
			const int stretch = (p.K + p.warps_k * STEP - 1) / (p.warps_k * STEP) * STEP, first = warp % p.warps_k * stretch, end = min(p.K, first + stretch);
			let_next_grid_start();
			wait_for_previous_grid();

			const T *rows[ROWS];
#pragma unroll
			for (int r = 0; r < ROWS; r++)
			{ // rows beyond the last: row 0 is read, and its sums go nowhere
				const int n = n0 + r % COLUMNS;
				rows[r] = p.w + static_cast<long long>(n < p.N ? n + (KIND == GATED && r >= COLUMNS ? p.N : 0) : 0) * p.K;
			}
			const T *tokens[TOKENS];
#pragma unroll
			for (int t = 0; t < TOKENS; t++) // beyond the last: the last again, without a branch between the loads
				tokens[t] = p.x + static_cast<long long>(min(t, p.tokens - 1)) * p.K;
			float acc[SUMS] = { }; // [row][token]
			auto multiply = [&](const Piece<T, VEC> (&w)[ROWS], int k)
			{
#pragma unroll
				for (int t = 0; t < TOKENS; t++)
				{
					const Piece<T, VEC> x = *reinterpret_cast<const Piece<T, VEC>*>(tokens[t] + k);
#pragma unroll
					for (int r = 0; r < ROWS; r++)
#pragma unroll
						for (int i = 0; i < VEC; i++)
							acc[r * TOKENS + t] = fmaf(to_float(w[r].v[i]), to_float(x.v[i]), acc[r * TOKENS + t]);
				}
			};
			if (n0 < p.N)
			{
				int k = first + lane * VEC;
				for (; k + (UNROLL - 1) * STEP < end; k += UNROLL * STEP)
				{
					Piece<T, VEC> w[UNROLL][ROWS];
#pragma unroll
					for (int i = 0; i < UNROLL; i++)
#pragma unroll
						for (int r = 0; r < ROWS; r++)
							w[i][r] = load_weights<T, VEC>(rows[r] + k + i * STEP);
#pragma unroll
					for (int i = 0; i < UNROLL; i++)
						multiply(w[i], k + i * STEP);
				}
				for (; k < end; k += STEP)
				{
					Piece<T, VEC> w[ROWS];
#pragma unroll
					for (int r = 0; r < ROWS; r++)
						w[r] = load_weights<T, VEC>(rows[r] + k);
					multiply(w, k);
				}
			}
			__syncwarp();
			sum_over_lanes<SUMS, 16>(acc, lane);
			constexpr int KEPT = SUMS > 32 ? SUMS / 32 : 1, SAME = SUMS < 32 ? 32 / SUMS : 1;
			if (lane % SAME == 0)
			{
#pragma unroll
				for (int i = 0; i < KEPT; i++)
					sums[warp][lane / SAME * KEPT + i] = acc[i];
			}
			__syncthreads();
			auto sum_of = [&](int group, int row, int t)
			{
				float s = 0.0f;
				for (int i = 0; i < p.warps_k; i++)
					s += sums[group * p.warps_k + i][row * TOKENS + t];
				return s;
			};
			if (KIND == STATISTICS)
			{ // a warp takes a token, a lane a column, or two
				constexpr int PER_LANE = (WARPS * COLUMNS + 31) / 32;
				for (int t = warp; t < p.tokens; t += WARPS)
				{
					float z[PER_LANE], top = -INFINITY, sum = 0.0f;
#pragma unroll
					for (int i = 0; i < PER_LANE; i++)
					{
						const int c = lane + i * 32, n = blockIdx.x * columns + c;
						const bool inside = c < columns && n < p.N;
						z[i] = inside ? sum_of(c / COLUMNS, c % COLUMNS, t) : -INFINITY;
						top = fmaxf(top, z[i]);
						if (inside && p.targets[t] == n)
							p.target_logit[t] = z[i];
					}
#pragma unroll
					for (int i = 16; i >= 1; i /= 2)
						top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
#pragma unroll
					for (int i = 0; i < PER_LANE; i++)
						sum += z[i] == -INFINITY ? 0.0f : expf(z[i] - top);
#pragma unroll
					for (int i = 16; i >= 1; i /= 2)
						sum += __shfl_xor_sync(0xffffffffu, sum, i);
					if (lane == 0)
						p.parts[static_cast<long long>(t) * gridDim.x + blockIdx.x] = make_float2(top, sum);
				}
				return;
			}
			for (int i = threadIdx.x; i < p.tokens * columns; i += WARPS * 32)
			{
				const int t = i / columns, c = i - t * columns, n = blockIdx.x * columns + c;
				if (n >= p.N)
					continue;
				T *dst = p.out + static_cast<long long>(t) * p.N + n;
				const float s = sum_of(c / COLUMNS, c % COLUMNS, t);
				if (KIND == GATED)
				{
					const float u = sum_of(c / COLUMNS, c % COLUMNS + COLUMNS, t);
					if (p.au != nullptr)
					{
						float *au = p.au + static_cast<long long>(t) * 2 * p.N + n;
						au[0] = s;
						au[p.N] = u;
					}
					*dst = from_float<T>(gate_by_code(p.gate, s) * u);
				}
				else
					*dst = from_float<T>(p.beta != 0.0f ? s + p.beta * to_float(*dst) : s);
			}
		}

		/* Warps that share a row: see above.  (GATED: N columns of the result are 2 N rows.) */
		int warps_along_k(mlContext_t ctx, int rows, int K, int tokens)
		{
			int warps_k = 1;
			while (warps_k < WARPS && rows / (WARPS / warps_k * rows_of_warp(tokens)) < 8 * get(ctx)->sm_count && K / (2 * warps_k) >= MIN_STRETCH)
				warps_k *= 2;
			return warps_k;
		}
		template<typename T, int VEC, int KIND>
		bool launch(mlContext_t ctx, const Params<T> &p)
		{
			const int columns = WARPS / p.warps_k * rows_of_warp(p.tokens) / (KIND == GATED ? 2 : 1);
			const dim3 grid((p.N + columns - 1) / columns), block(WARPS * 32);
			cudaStream_t stream = use_stream(ctx);
			const cudaError_t status = p.tokens == 1 ? launch_overlapped(kernel_few_rows<T, VEC, KIND, 1>, grid, block, 0, stream, p)
					: p.tokens == 2 ? launch_overlapped(kernel_few_rows<T, VEC, KIND, 2>, grid, block, 0, stream, p)
					: p.tokens <= 4 ? launch_overlapped(kernel_few_rows<T, VEC, KIND, 4>, grid, block, 0, stream, p)
					: p.tokens <= 8 ? launch_overlapped(kernel_few_rows<T, VEC, KIND, 8>, grid, block, 0, stream, p)
							: launch_overlapped(kernel_few_rows<T, VEC, KIND, 16>, grid, block, 0, stream, p);
			MB200_COUNT_LAUNCH();
			return check_cuda(ctx, status, "product of a few rows");
		}
		template<int KIND, typename T>
		bool launch(mlContext_t ctx, const FewRows<T> &f, Params<T> &p, int N)
		{
			p.tokens = f.tokens;
			p.K = f.K;
			p.N = N;
			p.warps_k = warps_along_k(ctx, KIND == GATED ? 2 * N : N, f.K, f.tokens);
			p.x = f.x;
			p.w = f.w;
			auto rows_aligned = [&](int elements)
			{
				return f.K % elements == 0 && aligned_to(f.x, elements * sizeof(T)) && aligned_to(f.w, elements * sizeof(T));
			};
			return rows_aligned(4) ? launch<T, 4, KIND>(ctx, p) : rows_aligned(2) ? launch<T, 2, KIND>(ctx, p) : launch<T, 1, KIND>(ctx, p);
		}
	}

	template<typename T>
	bool few_rows_gated(mlContext_t ctx, const FewRows<T> &f, int hidden, int gate, T *h, float *au)
	{
		Params<T> p = { };
		p.out = h;
		p.au = au;
		p.gate = gate;
		return launch<GATED>(ctx, f, p, hidden);
	}
	template<typename T>
	bool few_rows_product(mlContext_t ctx, const FewRows<T> &f, int N, T *y, float beta)
	{
		Params<T> p = { };
		p.out = y;
		p.beta = beta;
		return launch<PRODUCT>(ctx, f, p, N);
	}
	int few_rows_statistics_parts(mlContext_t ctx, int tokens, int N, int K)
	{
		const int columns = WARPS / warps_along_k(ctx, N, K, tokens) * rows_of_warp(tokens);
		return (N + columns - 1) / columns;
	}
	template<typename T>
	bool few_rows_statistics(mlContext_t ctx, const FewRows<T> &f, int N, const int *targets, float2 *parts, float *target_logit)
	{
		Params<T> p = { };
		p.targets = targets;
		p.parts = parts;
		p.target_logit = target_logit;
		return launch<STATISTICS>(ctx, f, p, N);
	}
	template bool few_rows_gated<__half>(mlContext_t, const FewRows<__half>&, int, int, __half*, float*);
	template bool few_rows_gated<float>(mlContext_t, const FewRows<float>&, int, int, float*, float*);
	template bool few_rows_product<__half>(mlContext_t, const FewRows<__half>&, int, __half*, float);
	template bool few_rows_product<float>(mlContext_t, const FewRows<float>&, int, float*, float);
	template bool few_rows_statistics<__half>(mlContext_t, const FewRows<__half>&, int, const int*, float2*, float*);
	template bool few_rows_statistics<float>(mlContext_t, const FewRows<float>&, int, const int*, float2*, float*);
} /* namespace mb200 */
