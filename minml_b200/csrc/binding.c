/*
 * binding.c -- the operators of transformer blocks as Python functions (module minml_b200._binding, used by backend.py).
 *
 * A layer norm's two calls for a few hundred rows are 11 us of kernels, and describing their sixteen tensors and passing them through ctypes was most
 * of 24 us of the host's time: a descriptor made in Python is five calls into torch, a packing and a copy.  Here the same five questions are asked
 * through the C API and the descriptors are passed as they are: 14 us.  A tensor that does not fit (another device, strides, rank) is handed to the function given to bind(), which
 * raises; afterwards the context's error, if any, is raised the same way.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>
#include <stdbool.h>
#include <string.h>

#include "minml_b200.h"

static PyObject *name_get_device, *name_is_contiguous, *name_shape, *name_dtype, *name_data_ptr;
static PyObject *dtype_codes, *refuse, *error_type; /* from bind() */
static struct
{
		__typeof__(&mb200_layernorm_forward) layernorm_forward;
		__typeof__(&mb200_layernorm_backward) layernorm_backward;
		__typeof__(&mb200_gated_feed_forward_forward) gated_feed_forward_forward;
		__typeof__(&mb200_gated_feed_forward_backward) gated_feed_forward_backward;
		__typeof__(&mb200_softmax_cross_entropy_forward) softmax_cross_entropy_forward;
		__typeof__(&mb200_softmax_cross_entropy_backward) softmax_cross_entropy_backward;
		__typeof__(&mb200_get_last_error) get_last_error;
		__typeof__(&mb200_clear_last_error) clear_last_error;
} library;

/* The value of an integer that a method of t returns; -2 and an exception if there is none. */
static long ask(PyObject *t, PyObject *method)
{
	PyObject *answer = PyObject_CallMethodNoArgs(t, method);
	if (answer == NULL)
		return -2;
	const long value = PyLong_AsLong(answer);
	Py_DECREF(answer);
	return value == -1 && PyErr_Occurred() ? -2 : value;
}
/* The shape of scratch memory says nothing but its size, so where an extent passes a descriptor's 32 bits it is described as rows of 256 elements (sizes asked
 * for are multiples of 256 bytes). */
#define SCRATCH_ROW 256
static bool describe(PyObject *t, PyObject *device, mlTensor_t *result, bool scratch)
{
	memset(result, 0, sizeof(*result));
	result->dtype = DTYPE_UNKNOWN;
	if (t == Py_None)
		return true;
	const long on = ask(t, name_get_device), wanted = PyLong_AsLong(device);
	if (PyErr_Occurred())
		return false;
	const long dense = ask(t, name_is_contiguous);
	if (dense == -2)
		return false;
	PyObject *shape = PyObject_GetAttr(t, name_shape);
	if (shape == NULL)
		return false;
	bool fits = on == wanted && dense == 1 && PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) <= 6;
	if (fits)
	{
		result->rank = (int) PyTuple_GET_SIZE(shape);
		long elements = 1; /* (of a tensor that exists, so the product fits) */
		bool long_extent = false;
		for (int i = 0; i < result->rank && fits; i++)
		{
			const long extent = PyLong_AsLong(PyTuple_GET_ITEM(shape, i));
			fits = extent >= 0 && (extent <= INT_MAX || scratch);
			long_extent |= extent > INT_MAX;
			elements *= extent;
			result->dim[i] = (int) extent;
		}
		if (fits && long_extent)
		{
			fits = elements / SCRATCH_ROW <= INT_MAX;
			memset(result->dim, 0, sizeof(result->dim));
			result->rank = 2;
			result->dim[0] = (int) (elements / SCRATCH_ROW);
			result->dim[1] = SCRATCH_ROW;
		}
	}
	Py_DECREF(shape);
	if (PyErr_Occurred())
		return false;
	if (!fits)
	{
		PyObject *none = PyObject_CallFunctionObjArgs(refuse, t, device, NULL);
		if (none != NULL)
		{
			Py_DECREF(none);
			PyErr_SetString(error_type, "a tensor that cannot be described");
		}
		return false;
	}
	PyObject *dtype = PyObject_GetAttr(t, name_dtype);
	if (dtype == NULL)
		return false;
	PyObject *code = PyDict_GetItemWithError(dtype_codes, dtype); /* borrowed */
	Py_DECREF(dtype);
	if (code != NULL)
		result->dtype = (mlDataType_t) PyLong_AsLong(code);
	PyObject *address = PyObject_CallMethodNoArgs(t, name_data_ptr);
	if (address == NULL)
		return false;
	result->data = PyLong_AsVoidPtr(address);
	Py_DECREF(address);
	return !PyErr_Occurred();
}

/* A call's arguments: the context's handle and device, `tensors` tensors or None, then `numbers` numbers. */
typedef struct
{
		mlContext_t context;
		mlTensor_t t[9];
		double number[3];
} Arguments;
enum Last
{
	RESULT, SCRATCH
}; /* what the last tensor is */
static bool take(Arguments *a, PyObject *const *args, Py_ssize_t given, int tensors, enum Last last, int numbers)
{
	if (given != 2 + tensors + numbers)
	{
		PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", 2 + tensors + numbers, given);
		return false;
	}
	if (library.get_last_error == NULL)
	{
		PyErr_SetString(PyExc_RuntimeError, "bind() has not been called");
		return false;
	}
	a->context = args[0] == Py_None ? NULL : PyLong_AsVoidPtr(args[0]);
	if (PyErr_Occurred())
		return false;
	for (int i = 0; i < tensors; i++)
		if (!describe(args[2 + i], args[1], &a->t[i], last == SCRATCH && i == tensors - 1))
			return false;
	for (int i = 0; i < numbers; i++)
	{
		a->number[i] = PyFloat_AsDouble(args[2 + tensors + i]);
		if (PyErr_Occurred())
			return false;
	}
	return true;
}
static PyObject* outcome(const Arguments *a)
{
	const char *message = library.get_last_error(a->context);
	if (message == NULL || message[0] == '\0')
		Py_RETURN_NONE;
	PyErr_SetString(error_type, message);
	library.clear_last_error(a->context);
	return NULL;
}

static PyObject* layernorm_forward(PyObject *self, PyObject *const *args, Py_ssize_t given)
{
	Arguments a;
	if (!take(&a, args, given, 6, RESULT, 0))
		return NULL;
	Py_BEGIN_ALLOW_THREADS
	library.layernorm_forward(a.context, a.t[0], a.t[1], a.t[2], a.t[3], a.t[4], a.t[5]);
	Py_END_ALLOW_THREADS
	return outcome(&a);
}
static PyObject* layernorm_backward(PyObject *self, PyObject *const *args, Py_ssize_t given)
{
	Arguments a;
	if (!take(&a, args, given, 9, SCRATCH, 2))
		return NULL;
	Py_BEGIN_ALLOW_THREADS
	library.layernorm_backward(a.context, a.t[0], a.t[1], a.t[2], a.t[3], a.t[4], (float) a.number[0], a.t[5], (float) a.number[1], a.t[6], a.t[7], a.t[8]);
	Py_END_ALLOW_THREADS
	return outcome(&a);
}
static PyObject* gated_feed_forward_forward(PyObject *self, PyObject *const *args, Py_ssize_t given)
{
	Arguments a;
	if (!take(&a, args, given, 6, SCRATCH, 2))
		return NULL;
	Py_BEGIN_ALLOW_THREADS
	library.gated_feed_forward_forward(a.context, a.t[0], a.t[1], a.t[2], (float) a.number[0], a.t[3], (int) a.number[1], a.t[4], a.t[5]);
	Py_END_ALLOW_THREADS
	return outcome(&a);
}
static PyObject* gated_feed_forward_backward(PyObject *self, PyObject *const *args, Py_ssize_t given)
{
	Arguments a;
	if (!take(&a, args, given, 9, SCRATCH, 3))
		return NULL;
	Py_BEGIN_ALLOW_THREADS
	library.gated_feed_forward_backward(a.context, a.t[0], a.t[1], a.t[2], a.t[3], a.t[4], (float) a.number[0], a.t[5], (float) a.number[1], a.t[6], a.t[7], (int) a.number[2], a.t[8]);
	Py_END_ALLOW_THREADS
	return outcome(&a);
}
static PyObject* softmax_cross_entropy_forward(PyObject *self, PyObject *const *args, Py_ssize_t given)
{
	Arguments a;
	if (!take(&a, args, given, 6, SCRATCH, 0))
		return NULL;
	Py_BEGIN_ALLOW_THREADS
	library.softmax_cross_entropy_forward(a.context, a.t[0], a.t[1], a.t[2], a.t[3], a.t[4], a.t[5]);
	Py_END_ALLOW_THREADS
	return outcome(&a);
}
static PyObject* softmax_cross_entropy_backward(PyObject *self, PyObject *const *args, Py_ssize_t given)
{
	Arguments a;
	if (!take(&a, args, given, 8, SCRATCH, 3))
		return NULL;
	Py_BEGIN_ALLOW_THREADS
	library.softmax_cross_entropy_backward(a.context, a.t[0], a.t[1], a.t[2], a.t[3], (float) a.number[0], a.t[4], (float) a.number[1], a.t[5], (float) a.number[2], a.t[6], a.t[7]);
	Py_END_ALLOW_THREADS
	return outcome(&a);
}

/* bind(addresses of the library's functions by name, codes by dtype, function that raises for a tensor and a device, exception type) */
static PyObject* bind(PyObject *self, PyObject *args)
{
	PyObject *addresses, *codes, *raises, *type;
	if (!PyArg_ParseTuple(args, "O!O!OO", &PyDict_Type, &addresses, &PyDict_Type, &codes, &raises, &type))
		return NULL;
	const struct
	{
			const char *name;
			void *function;
	} wanted[] = { { "mb200_layernorm_forward", &library.layernorm_forward }, { "mb200_layernorm_backward", &library.layernorm_backward }, { "mb200_gated_feed_forward_forward",
			&library.gated_feed_forward_forward }, { "mb200_gated_feed_forward_backward", &library.gated_feed_forward_backward }, { "mb200_softmax_cross_entropy_forward",
			&library.softmax_cross_entropy_forward }, { "mb200_softmax_cross_entropy_backward", &library.softmax_cross_entropy_backward }, { "mb200_clear_last_error",
			&library.clear_last_error }, { "mb200_get_last_error", &library.get_last_error } };
	for (size_t i = 0; i < sizeof(wanted) / sizeof(wanted[0]); i++)
	{
		PyObject *address = PyDict_GetItemString(addresses, wanted[i].name);
		void *p = address == NULL ? NULL : PyLong_AsVoidPtr(address);
		if (p == NULL)
		{
			if (!PyErr_Occurred())
				PyErr_Format(PyExc_KeyError, "%s", wanted[i].name);
			return NULL;
		}
		memcpy(wanted[i].function, &p, sizeof(p));
	}
	Py_XSETREF(dtype_codes, Py_NewRef(codes));
	Py_XSETREF(refuse, Py_NewRef(raises));
	Py_XSETREF(error_type, Py_NewRef(type));
	Py_RETURN_NONE;
}

#define FAST(name) { #name, (PyCFunction) (void (*)(void)) name, METH_FASTCALL, NULL }
static PyMethodDef methods[] = { { "bind", bind, METH_VARARGS, NULL }, FAST(layernorm_forward), FAST(layernorm_backward), FAST(gated_feed_forward_forward),
		FAST(gated_feed_forward_backward), FAST(softmax_cross_entropy_forward), FAST(softmax_cross_entropy_backward), { NULL, NULL, 0, NULL } };
static struct PyModuleDef module = { .m_base = PyModuleDef_HEAD_INIT, .m_name = "_binding", .m_size = -1, .m_methods = methods };

PyMODINIT_FUNC PyInit__binding(void)
{
	name_get_device = PyUnicode_InternFromString("get_device");
	name_is_contiguous = PyUnicode_InternFromString("is_contiguous");
	name_shape = PyUnicode_InternFromString("shape");
	name_dtype = PyUnicode_InternFromString("dtype");
	name_data_ptr = PyUnicode_InternFromString("data_ptr");
	return name_get_device == NULL || name_is_contiguous == NULL || name_shape == NULL || name_dtype == NULL || name_data_ptr == NULL ? NULL : PyModule_Create(&module);
}
