/*
 * gemm_fp32.cuh -- the fp32 products of the feed-forward and loss operators, and the copies that give an operand a pitch TMA can address.
 */
#pragma once

#include "common.cuh"

namespace mb200
{
	/* As PairOperand (gemm_pair.cuh), of fp32. */
	struct FloatOperand
	{
			const void *data = nullptr;
			int ld = 0;
			bool mn = false;
	};
	/* D = A B^T + beta D, fp32; `partials` holds float_partial_elements(M, N, K) floats. */
	size_t float_partial_elements(mlContext_t ctx, int M, int N, int K);
	bool float_product(mlContext_t ctx, int M, int N, int K, const FloatOperand &a, const FloatOperand &b, float *d, int ldd, float beta, float *partials);

	/* dst [blocks * padded_rows, pitch] = src [blocks * rows, columns], the added rows and columns zero */
	template<typename T>
	bool pack_rows(mlContext_t ctx, T *dst, int pitch, long long padded_rows, const T *src, long long rows, int columns, int blocks = 1);
} /* namespace mb200 */
