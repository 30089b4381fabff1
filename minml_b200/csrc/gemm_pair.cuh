/*
 * gemm_pair.cuh -- interface of the fp16 products of the feed-forward and loss operators (gemm_pair.cu): A (M x K) times B^T (N x K), fp32
 * accumulators, with the operator's next step in the epilogue.
 */
#pragma once

#include "common.cuh"

namespace mb200
{
	/* An operand of `rows` (M or N) by K, stored [rows, K] (mn = false) or [K, rows] (mn = true), `ld` elements from row to row.  TMA reads it:
	 * 16-byte aligned base and row pitch. */
	struct PairOperand
	{
			const void *data = nullptr;
			int ld = 0;
			bool mn = false;
	};
	/* D[m, n] = alpha * alpha_device * row_scale[m] * sum + beta * D, one rounding to fp16; the optional factors are 1 when null, a row of
	 * scale 0 is 0 whatever its sum. */
	struct PairResult
	{
			__half *d = nullptr;
			int ldd = 0;
			float alpha = 1.0f, beta = 0.0f;
			const float *alpha_device = nullptr;
			const float *row_scale = nullptr;
	};

	/* Number of K ranges a product is best cut into (1: none), and the fp32 scratch its partial results need. */
	int pair_splits(mlContext_t ctx, int M, int N, int K);
	size_t pair_partial_elements(mlContext_t ctx, int M, int N, int K); // 0 when the product is not cut
	/* D = A B^T; `partials` as large as pair_partial_elements says. */
	bool pair_product(mlContext_t ctx, int M, int N, int K, const PairOperand &a, const PairOperand &b, const PairResult &r, float *partials);

	/* sums[s] (M x pitch floats each) = or += the product of K range s of `splits`; finish_sums adds them up into a result. */
	bool pair_product_sums(mlContext_t ctx, int M, int N, int K, const PairOperand &a, const PairOperand &b, float *sums, int pitch, int splits, bool accumulate);
	template<typename T>
	bool finish_sums(mlContext_t ctx, T *d, int ldd, int M, int N, const float *sums, int pitch, int splits, float alpha, const float *alpha_device, const float *row_scale, float beta);

	/* h = act(a) u with a = x Wg^T, u = x Wu^T, w1 = [Wg; Wu] (2 hidden rows).  h [tokens, hidden], pitch ldh (a multiple of 8 elements, 16-byte
	 * aligned).  kept: null, or 2 tokens hidden floats that receive a and u, in an order of this kernel's own (hidden a multiple of 4). */
	bool pair_gated(mlContext_t ctx, int tokens, int embed, int hidden, const PairOperand &x, const PairOperand &w1, int gate, __half *h, int ldh, float *kept);
	/* From dh = dy W2 and what pair_gated kept: dau = [dh u act'(a), dh act(a)] fp16 [tokens, 2 hidden], h = act(a) u fp16 [tokens, hidden]; hidden a
	 * multiple of 8. */
	bool pair_gated_backward(mlContext_t ctx, int tokens, int embed, int hidden, const PairOperand &dy, const PairOperand &w2, int gate, const float *kept, __half *dau, __half *h);

	/* The same with nothing kept: a and u are made again, in the same tiles as dh; h may be null (not wanted).  dy [tokens, embed] and w2 stored [embed, hidden] (mn). */
	bool pair_gated_recompute(mlContext_t ctx, int tokens, int embed, int hidden, const PairOperand &x, const PairOperand &w1, const PairOperand &dy, const PairOperand &w2, int gate, __half *dau,
			__half *h);

	/* Row statistics of the logits x w^T over columns first .. first + N: parts[t][i] = (maximum, sum of exp(z - maximum)) of group i of
	 * 128 columns, pair_statistics_parts(N) groups; target_logit[t] where the row's target lies in the range. */
	int pair_statistics_parts(int N);
	bool pair_statistics(mlContext_t ctx, int tokens, int N, int embed, const PairOperand &x, const PairOperand &w, const int *targets, float2 *parts, float *target_logit);
	/* p = 2^15 (exp(z - lse) - [column = target]) fp16, pitch ldp, for columns first .. first + N of the vocabulary; 0 in the rows with a target outside
	 * [0, vocab) or a weight of 0. */
	bool pair_probabilities(mlContext_t ctx, int tokens, int N, int embed, const PairOperand &x, const PairOperand &w, const int *targets, const float *row_weights, const float *lse, int first,
			int vocab, __half *p, int ldp);
} /* namespace mb200 */
