/*
 * few_rows.cuh -- products of a few rows with a large weight matrix on the fp32 units (few_rows.cu): fp32 data, and fp16 data whose rows do
 * not start on 16-byte boundaries.  Everything is dense: pitches are the row lengths, and pointers need no more than their elements' alignment.
 */
#pragma once

#include "common.cuh"

namespace mb200
{
	/* Rows up to which they are the faster way.  fp32, against gemm_fp32.cu: 16 rows, V = 50021, embed 2048: 161 us to 209, embed 2049: 222 to 341;
	 * the kernels take no more.  fp16, against few_tokens.cu and the copies it needs: embed 4097, hidden 11009: 8 rows 135 us, 9 rows 263 to 179. */
	constexpr int FEW_ROWS_FP32 = 16, FEW_ROWS_FP16 = 8;

	template<typename T>
	struct FewRows
	{
			int tokens, K;
			const T *x; // [tokens, K]
			const T *w; // [rows, K]
	};
	/* h [tokens, hidden] = act(a) u, w = [Wg; Wu]; au: null, or fp32 [tokens, 2 hidden] that receives a and u */
	template<typename T>
	bool few_rows_gated(mlContext_t ctx, const FewRows<T> &p, int hidden, int gate, T *h, float *au);
	/* y [tokens, N] = x w^T + beta y */
	template<typename T>
	bool few_rows_product(mlContext_t ctx, const FewRows<T> &p, int N, T *y, float beta);
	/* As pair_statistics (gemm_pair.cuh), with few_rows_statistics_parts(ctx, tokens, N, K) groups of columns */
	int few_rows_statistics_parts(mlContext_t ctx, int tokens, int N, int K);
	template<typename T>
	bool few_rows_statistics(mlContext_t ctx, const FewRows<T> &p, int N, const int *targets, float2 *parts, float *target_logit);
} /* namespace mb200 */
