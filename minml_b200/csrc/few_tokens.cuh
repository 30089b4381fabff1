/*
 * few_tokens.cuh -- fp16 products of at most 64 rows with a large weight matrix (few_tokens.cu): decoding, scoring of a few tokens.
 */
#pragma once

#include "common.cuh"

namespace mb200
{
	constexpr int FEW_TOKENS = 64;

	/* Rows of `embed` (x, and w row-major [rows, embed]) with pitches ldx, ldw that are multiples of 8 elements from 16-byte aligned bases. */
	struct FewTokens
	{
			int tokens, embed;
			const __half *x;
			int ldx;
			const __half *w;
			int ldw;
	};
	/* h = act(a) u, w = [Wg; Wu]; h has pitch ldh and ldh - hidden columns of padding that are left as they are */
	bool few_gated(mlContext_t ctx, const FewTokens &p, int hidden, int gate, __half *h, int ldh);
	/* y [tokens, N] = x w^T + beta y.  The launch ahead of this one in the stream has to be few_gated's: the first weights are fetched under it. */
	bool few_product_after_gated(mlContext_t ctx, const FewTokens &p, int N, __half *y, int ldy, float beta);
	/* As pair_statistics (gemm_pair.cuh), with few_statistics_parts(ctx, N) groups of columns */
	int few_statistics_parts(mlContext_t ctx, int N);
	bool few_statistics(mlContext_t ctx, const FewTokens &p, int N, const int *targets, float2 *parts, float *target_logit);
} /* namespace mb200 */
