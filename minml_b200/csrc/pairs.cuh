/*
 * pairs.cuh -- arithmetic on two fp32 values at a time: sm_100a multiplies and adds register pairs in one instruction.
 */
#pragma once

#include "common.cuh"

namespace mb200
{
	struct Pair
	{
			float x, y;
	};
	__device__ __forceinline__ Pair pair_fma(Pair a, Pair b, Pair c)
	{
		Pair d;
		asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
				: "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
		return d;
	}
	__device__ __forceinline__ Pair pair_mul(Pair a, Pair b)
	{
		Pair d;
		asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
				: "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
		return d;
	}
	__device__ __forceinline__ Pair pair_add(Pair a, Pair b)
	{
		Pair d;
		asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
				: "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
		return d;
	}
	__device__ __forceinline__ Pair pair_of(float v)
	{
		return Pair { v, v };
	}
} /* namespace mb200 */
