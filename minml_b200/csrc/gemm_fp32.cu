/*
 * gemm_fp32.cu -- see gemm_fp32.cuh.
 */
#include "common.cuh"
#include "gemm.cuh"
#include "gemm_fp32.cuh"

#include <algorithm>

namespace mb200
{
	namespace
	{
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_pack_rows(T *__restrict__ dst, int pitch, long long padded_rows, const T *__restrict__ src, long long rows, int columns, int blocks)
		{
			for (long long r = blockIdx.x; r < padded_rows * blocks; r += gridDim.x)
			{
				const long long block = r / padded_rows, inside = r - block * padded_rows;
				const T *from = src + (block * rows + inside) * columns;
				for (int c = threadIdx.x; c < pitch; c += 256)
					dst[r * pitch + c] = inside < rows && c < columns ? from[c] : from_float<T>(0.0f);
			}
		}
	}

	template<typename T>
	bool pack_rows(mlContext_t ctx, T *dst, int pitch, long long padded_rows, const T *src, long long rows, int columns, int blocks)
	{
		const int grid = static_cast<int>(std::max<long long>(1, std::min<long long>(padded_rows * blocks, static_cast<long long>(get(ctx)->sm_count) * 8)));
		kernel_pack_rows<T> <<<grid, 256, 0, use_stream(ctx)>>>(dst, pitch, padded_rows, src, rows, columns, blocks);
		MB200_COUNT_LAUNCH();
		return check_cuda(ctx, cudaGetLastError(), "pack_rows");
	}
	template bool pack_rows<__half>(mlContext_t, __half*, int, long long, const __half*, long long, int, int);
	template bool pack_rows<float>(mlContext_t, float*, int, long long, const float*, long long, int, int);

	bool float_product(mlContext_t ctx, int M, int N, int K, const FloatOperand &a, const FloatOperand &b, float *d, int ldd, float alpha, float beta)
	{
		GemmTcProblem g;
		g.kind = 3;
		g.M = M;
		g.N = N;
		g.K = K;
		g.a_mn = a.mn;
		g.b_mn = b.mn;
		g.A = a.data;
		g.lda = a.ld;
		g.B = b.data;
		g.ldb = b.ld;
		g.D = d;
		g.ldd = ldd;
		g.C = d;
		g.ldc = ldd;
		g.alpha = alpha;
		g.beta = beta;
		g.out_dtype = DTYPE_FLOAT32;
		return gemm_tc_run(ctx, g);
	}
} /* namespace mb200 */
