/*
 * operands.cuh -- host-side checks of descriptor arguments, shared by the entry points of the training operators
 * (layernorm_train.cu, feed_forward.cu, cross_entropy.cu).  A failed check records the sticky error and returns false.
 */
#pragma once

#include "common.cuh"

#include <initializer_list>

namespace mb200
{
	inline bool is_empty_descriptor(const mlTensor_t &t)
	{
		return t.data == nullptr && t.rank == 0;
	}
	inline const char* dtype_name(mlDataType_t dtype)
	{
		switch (dtype)
		{
			case DTYPE_FLOAT16:
				return "fp16";
			case DTYPE_FLOAT32:
				return "fp32";
			case DTYPE_FLOAT64:
				return "fp64";
			case DTYPE_INT32:
				return "int32";
			case DTYPE_UINT8:
				return "uint8";
			default:
				return "another type";
		}
	}
	/* Rows and columns of a matrix at most: the kernels' 32-bit indices pass the end by less than 4096 (a tile, the step of a loop). */
	constexpr long long MAX_EXTENT = 0x7FFFF000;
	/* A rank within the descriptor's array, no negative extent and a volume of 64 bits in bytes: what every later use of dim[] relies on. */
	inline bool check_extents(mlContext_t ctx, const char *who, const char *name, const mlTensor_t &t)
	{
		if (t.rank < 1 || t.rank > 6)
		{
			record_error(ctx, "%s: %s has rank %d", who, name, t.rank);
			return false;
		}
		for (int i = 0; i < t.rank; i++)
			if (t.dim[i] < 0)
			{
				record_error(ctx, "%s: %s has a negative extent", who, name);
				return false;
			}
		long long elements = 1;
		for (int i = 0; i < t.rank && elements != 0; i++)
		{
			if (t.dim[i] > 0 && elements > (1ll << 59) / t.dim[i])
			{
				record_error(ctx, "%s: %s has more elements than any memory", who, name);
				return false;
			}
			elements *= t.dim[i];
		}
		return true;
	}
	/* `t` holds rows x columns elements of `dtype`: a matrix whose leading extents multiply to `rows` and whose last is `columns`, or, for
	 * columns < 0, any shape of `rows` elements in all.  An empty tensor may have null data. */
	inline bool check_operand(mlContext_t ctx, const char *who, const char *name, const mlTensor_t &t, mlDataType_t dtype, long long rows, long long columns = -1)
	{
		if (!check_extents(ctx, who, name, t))
			return false;
		if (t.dtype != dtype)
		{
			record_error(ctx, "%s: %s is %s, expected %s", who, name, dtype_name(t.dtype), dtype_name(dtype));
			return false;
		}
		const long long wanted = columns < 0 ? rows : rows * columns;
		if (volume(t) != wanted || (columns >= 0 && last_dim(t) != columns))
		{
			if (columns < 0)
				record_error(ctx, "%s: %s has %lld elements, expected %lld", who, name, volume(t), rows);
			else
				record_error(ctx, "%s: %s has %lld elements in rows of %d, expected %lld rows of %lld", who, name, volume(t), last_dim(t), rows, columns);
			return false;
		}
		if (wanted > 0 && (t.data == nullptr || !aligned_to(t.data, size_of(dtype))))
		{
			record_error(ctx, "%s: %s is null or not aligned to its element size", who, name);
			return false;
		}
		return true;
	}
	inline long long bytes_of(const mlTensor_t &t)
	{
		return volume(t) * size_of(t.dtype);
	}
	/* The result `out` may be the very same memory as an input where `in_place` allows it, never a part of it. */
	inline bool check_distinct(mlContext_t ctx, const char *who, const char *out_name, const mlTensor_t &out, const char *in_name, const mlTensor_t &in, bool in_place = false)
	{
		if (out.data == nullptr || in.data == nullptr || bytes_of(out) == 0 || bytes_of(in) == 0 || !ranges_overlap(out.data, bytes_of(out), in.data, bytes_of(in)))
			return true;
		if (in_place && out.data == in.data && bytes_of(out) == bytes_of(in))
			return true;
		record_error(ctx, "%s: %s overlaps %s", who, out_name, in_name);
		return false;
	}
	inline bool check_workspace(mlContext_t ctx, const char *who, const mlTensor_t &workspace, size_t needed)
	{
		if (needed == 0)
			return true;
		if (is_empty_descriptor(workspace) || workspace.data == nullptr)
		{
			record_error(ctx, "%s: needs a workspace of %zu bytes", who, needed);
			return false;
		}
		if (!check_extents(ctx, who, "workspace", workspace))
			return false;
		if (bytes_of(workspace) < static_cast<long long>(needed) || !aligned_to(workspace.data, 16))
		{
			record_error(ctx, "%s: the workspace has %lld bytes (16-byte aligned: %s), %zu are needed", who, bytes_of(workspace),
					aligned_to(workspace.data, 16) ? "yes" : "no", needed);
			return false;
		}
		return true;
	}
	/* Hands out 256-byte aligned pieces of a workspace; `used` is also the size that a run with a null base asks for. */
	struct Carver
	{
			uint8_t *base;
			size_t used = 0;
			explicit Carver(void *workspace) :
					base(reinterpret_cast<uint8_t*>(workspace))
			{
			}
			template<typename T>
			T* take(size_t elements)
			{
				T *result = base == nullptr ? nullptr : reinterpret_cast<T*>(base + used);
				used += (elements * sizeof(T) + 255) / 256 * 256;
				return result;
			}
	};
	inline int round_up(int n, int to)
	{
		return (n + to - 1) / to * to;
	}
	inline mlTensor_t no_tensor()
	{
		mlTensor_t t = { };
		return t;
	}
	/* Walks a grid over rows x groups: a 64-bit division by a run-time number is dozens of instructions, so up to 2^31 places go by FastDiv. */
	struct GridWalk
	{
			long long total;
			long long groups;
			FastDiv by_groups;
			int small;
			GridWalk() = default;
			GridWalk(long long rows, long long groups_of_row) :
					total(rows * groups_of_row),
					groups(groups_of_row),
					by_groups(static_cast<uint32_t>(groups_of_row <= 0x7FFFFFFFll ? groups_of_row : 1)),
					small(total <= 0x7FFFFFFFll)
			{
			}
			__device__ __forceinline__ void place(long long i, long long &row, int &group) const
			{
				if (small)
				{
					uint32_t q, r;
					by_groups.divmod(static_cast<uint32_t>(i), q, r);
					row = q;
					group = static_cast<int>(r);
				}
				else
				{
					row = i / groups;
					group = static_cast<int>(i - row * groups);
				}
			}
	};
	/* Launch whose grid may start before the grid ahead of it in the stream has finished; the kernel calls griddepcontrol.wait
	 * (wait_for_previous_grid) before it touches anything that grid wrote, and reads through pointers without __restrict__ and without __ldg:
	 * both promise memory that nobody writes during the kernel, which is read through a path that is not coherent and may be read ahead of the
	 * wait. */
	template<typename ... KArgs, typename ... Args>
	inline cudaError_t launch_overlapped(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args ... args)
	{
		cudaLaunchConfig_t config = { };
		config.gridDim = grid;
		config.blockDim = block;
		config.dynamicSmemBytes = smem;
		config.stream = stream;
		cudaLaunchAttribute attribute = { };
		attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
		attribute.val.programmaticStreamSerializationAllowed = 1;
		config.attrs = &attribute;
		config.numAttrs = 1;
		return cudaLaunchKernelEx(&config, kernel, static_cast<KArgs>(args)...);
	}
	__device__ __forceinline__ void wait_for_previous_grid()
	{
		asm volatile("griddepcontrol.wait;" ::: "memory");
	}
	/* Without this a dependent grid starts only when this one ends; its writes are visible after wait_for_previous_grid either way. */
	__device__ __forceinline__ void let_next_grid_start()
	{
		asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
	}
} /* namespace mb200 */
