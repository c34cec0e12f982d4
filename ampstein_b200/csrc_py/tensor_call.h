/* Calls of the attention operators that take torch tensors as they are: the checks that attention.py makes in some hundred
 * Python steps (8 to 12 us of a call that takes the device 3), made here on the tensors' descriptions (DLPack's exchange interface, which
 * torch offers as a table of C functions; without one these calls do not exist, and attention.py does its own checks).
 * A call returns None when anything is not as usual (another type, a tensor of another device, a shape that does not fit, an
 * error of the entry): attention.py then goes its own way, which says what is wrong. Nothing has been launched then, except by an
 * entry that failed itself. */
#if defined(__has_include)
#if __has_include(<ATen/dlpack.h>)
#include <ATen/dlpack.h>
#endif
#endif

#if defined(DLPACK_MAJOR_VERSION) && DLPACK_MAJOR_VERSION == 1 && DLPACK_MINOR_VERSION >= 3
#define TENSOR_CALLS 1

static const DLPackExchangeAPI* tc_api;
static PyTypeObject* tc_type;

/* tensor_setup(torch.Tensor): whether the calls below work */
ENTRY(tensor_setup)
{
    PyObject* cap;
    if (!count("tensor_setup", n, 1)) return NULL;
    if (!PyType_Check(a[0])) Py_RETURN_FALSE;
    cap = PyObject_GetAttrString(a[0], "__dlpack_c_exchange_api__");
    if (cap)
    {
        const DLPackExchangeAPI* t = (const DLPackExchangeAPI*) PyCapsule_GetPointer(cap, "dlpack_exchange_api");
        if (t && t->header.version.major == 1 && t->dltensor_from_py_object_no_sync && t->current_work_stream)
        {
            Py_INCREF(a[0]);
            tc_type = (PyTypeObject*) a[0];
            tc_api = t;
        }
        Py_DECREF(cap);
    }
    PyErr_Clear();
    if (tc_api) Py_RETURN_TRUE;
    Py_RETURN_FALSE;
}

/* a CUDA tensor on device `dev` (-1: any) */
static int tc_get(PyObject* o, DLTensor* t, int dev)
{
    if (!tc_api || Py_TYPE(o) != tc_type) return 0;
    if (tc_api->dltensor_from_py_object_no_sync(o, t)) { PyErr_Clear(); return 0; }
    return t->device.device_type == kDLCUDA && (dev < 0 || t->device.device_id == dev) && t->dtype.lanes == 1;
}

static char* tc_ptr(const DLTensor* t) { return t->data ? (char*) t->data + t->byte_offset : NULL; }
static int tc_is(const DLTensor* t, int code, int bits) { return t->dtype.code == code && t->dtype.bits == bits; }
static int tc_same(const DLTensor* t, const DLTensor* u) { return t->dtype.code == u->dtype.code && t->dtype.bits == u->dtype.bits; }
static long tc_stride(const DLTensor* t, int d) { return t->shape[d] > 1 ? (long) t->strides[d] : 0; }
static int tc_dense(const DLTensor* t, int d) { return t->shape[d] <= 1 || t->strides[d] == 1; }
static int tc_fits(int64_t v) { return v >= 0 && v <= 0x7fffffff; }

static int tc_half(const DLTensor* t, int* bf16)
{
    *bf16 = tc_is(t, kDLBfloat, 16);
    return *bf16 || tc_is(t, kDLFloat, 16);
}

/* (rows, heads, dim) */
static int tc_rows(const DLTensor* t) { return t->ndim == 3 && tc_dense(t, 2) && tc_fits(t->shape[0]) && tc_fits(t->shape[1]) && tc_fits(t->shape[2]); }
static int tc_shape(const DLTensor* t, int64_t a, int64_t b, int64_t c) { return t->shape[0] == a && t->shape[1] == b && t->shape[2] == c; }

static int tc_cache(const DLTensor* t, int64_t kv_heads, int64_t dim)
{
    return t->ndim == 4 && tc_dense(t, 3) && t->shape[2] == kv_heads && t->shape[3] == dim && t->shape[0] >= 1 && t->shape[1] >= 1 &&
           tc_fits(t->shape[0]) && tc_fits(t->shape[1]);
}

/* no stride inside the extent of a smaller one: every place of what is written is its own */
static int tc_apart(const DLTensor* t)
{
    int64_t extent = 1;
    int done[8] = { 0 }, d, k;
    if (t->ndim > 8) return 0;
    for (k = 0; k < t->ndim; ++k)
    {
        int best = -1;
        for (d = 0; d < t->ndim; ++d) if (!done[d] && t->shape[d] > 1 && (best < 0 || t->strides[d] < t->strides[best])) best = d;
        if (best < 0) return 1;
        if (t->strides[best] < extent) return 0;
        extent += t->strides[best] * (t->shape[best] - 1);
        done[best] = 1;
    }
    return 1;
}

/* pos and cu (None) of `rows` rows */
static int tc_sequences(PyObject* pos_o, PyObject* cu_o, int64_t rows, int dev, const void** pos, const int** cu, int* seqs, int* pos64)
{
    DLTensor p, c;
    if (!tc_get(pos_o, &p, dev) || p.ndim != 1 || !tc_dense(&p, 0) || p.dtype.code != kDLInt || (p.dtype.bits != 32 && p.dtype.bits != 64) ||
        p.shape[0] < 1 || !tc_fits(p.shape[0])) return 0;
    *pos = tc_ptr(&p); *seqs = (int) p.shape[0]; *pos64 = p.dtype.bits == 64; *cu = NULL;
    if (cu_o == Py_None) return rows % *seqs == 0;
    if (!tc_get(cu_o, &c, dev) || c.ndim != 1 || !tc_dense(&c, 0) || !tc_is(&c, kDLInt, 32) || c.shape[0] != p.shape[0] + 1) return 0;
    *cu = (const int*) tc_ptr(&c);
    return 1;
}

static int tc_table(PyObject* o, int seqs, int64_t page_size, int dev, const int** table, long* row, int* max_pages)
{
    DLTensor t;
    if (!tc_get(o, &t, dev) || t.ndim != 2 || t.shape[0] != seqs || !tc_dense(&t, 1) || !tc_is(&t, kDLInt, 32) || t.shape[1] > (1 << 30) / page_size) return 0;
    *table = (const int*) tc_ptr(&t); *row = tc_stride(&t, 0); *max_pages = (int) t.shape[1];
    return 1;
}

/* the current device's number and its torch stream; 0: the tensors are on another device */
static int tc_stream(int dev, cudaStream_t* st)
{
    int cur = -1;
    void* s = NULL;
    if (cudaGetDevice(&cur) != cudaSuccess || cur != dev) return 0;
    if (tc_api->current_work_stream(kDLCUDA, dev, &s)) { PyErr_Clear(); return 0; }
    *st = (cudaStream_t) s;
    return 1;
}

#define TC_RUN(expr) do { int rc; Py_BEGIN_ALLOW_THREADS rc = (expr); Py_END_ALLOW_THREADS if (rc) Py_RETURN_NONE; return PyLong_FromLong(0); } while (0)

/* rope_call(q, k, v, pos, inv_freq, k_cache, v_cache, table, cu, interleaved, mscale, out); k None: q alone */
ENTRY(rope_call)
{
    amp_rope_args P;
    DLTensor q, k, v, f, kc, vc, out;
    cudaStream_t st;
    int dev, truth;
    double mscale;
    if (!count("rope_call", n, 12)) return NULL;
    memset(&P, 0, sizeof P);
    if (!tc_get(a[0], &q, -1) || !tc_rows(&q) || !tc_half(&q, &P.bf16) || q.shape[0] < 1) Py_RETURN_NONE;
    dev = q.device.device_id;
    if (!tc_get(a[11], &out, dev) || !tc_rows(&out) || !tc_same(&out, &q) || !tc_shape(&out, q.shape[0], q.shape[1], q.shape[2]) || !tc_apart(&out)) Py_RETURN_NONE;
    if (!tc_get(a[4], &f, dev) || f.ndim != 1 || !tc_dense(&f, 0) || !tc_is(&f, kDLFloat, 32) || 2 * f.shape[0] > q.shape[2]) Py_RETURN_NONE;
    if (!tc_sequences(a[3], a[8], q.shape[0], dev, &P.pos, &P.cu, &P.seqs, &P.pos64)) Py_RETURN_NONE;
    P.q = tc_ptr(&q); P.q_out = tc_ptr(&out); P.inv_freq = (const float*) tc_ptr(&f);
    P.q_token = tc_stride(&q, 0); P.q_head = tc_stride(&q, 1); P.out_token = tc_stride(&out, 0); P.out_head = tc_stride(&out, 1);
    if (P.q == P.q_out && (P.q_token != P.out_token || P.q_head != P.out_head)) Py_RETURN_NONE;
    P.tokens = (int) q.shape[0]; P.heads = (int) q.shape[1]; P.dim = (int) q.shape[2]; P.rot = 2 * (int) f.shape[0];
    truth = PyObject_IsTrue(a[9]);
    mscale = PyFloat_AsDouble(a[10]);
    if (truth < 0 || (mscale == -1.0 && PyErr_Occurred())) { PyErr_Clear(); Py_RETURN_NONE; }
    P.interleaved = truth; P.mscale = (float) mscale;
    if (a[1] != Py_None)
    {
        if (!tc_get(a[1], &k, dev) || !tc_rows(&k) || !tc_same(&k, &q) || k.shape[0] != q.shape[0] || k.shape[2] != q.shape[2]) Py_RETURN_NONE;
        if (!tc_get(a[2], &v, dev) || !tc_rows(&v) || !tc_same(&v, &q) || !tc_shape(&v, k.shape[0], k.shape[1], k.shape[2])) Py_RETURN_NONE;
        if (!tc_get(a[5], &kc, dev) || !tc_same(&kc, &q) || !tc_cache(&kc, k.shape[1], k.shape[2])) Py_RETURN_NONE;
        if (!tc_get(a[6], &vc, dev) || !tc_same(&vc, &q) || !tc_cache(&vc, k.shape[1], k.shape[2]) || vc.shape[0] != kc.shape[0] || vc.shape[1] != kc.shape[1] ||
            !tc_apart(&kc) || !tc_apart(&vc)) Py_RETURN_NONE;
        if (!tc_table(a[7], P.seqs, kc.shape[1], dev, &P.table, &P.table_row, &P.max_pages)) Py_RETURN_NONE;
        P.k = tc_ptr(&k); P.v = tc_ptr(&v); P.k_cache = tc_ptr(&kc); P.v_cache = tc_ptr(&vc);
        P.k_token = tc_stride(&k, 0); P.k_head = tc_stride(&k, 1); P.v_token = tc_stride(&v, 0); P.v_head = tc_stride(&v, 1);
        P.kc_page = tc_stride(&kc, 0); P.kc_row = tc_stride(&kc, 1); P.kc_head = tc_stride(&kc, 2);
        P.vc_page = tc_stride(&vc, 0); P.vc_row = tc_stride(&vc, 1); P.vc_head = tc_stride(&vc, 2);
        P.kv_heads = (int) k.shape[1]; P.pages = (int) kc.shape[0]; P.page_size = (int) kc.shape[1];
    }
    if (!tc_stream(dev, &st)) Py_RETURN_NONE;
    TC_RUN(amp_b200_rope(&P, st));
}

/* attention_call(q, k_cache, v_cache, table, pos, cu, window, sinks, scale, out, lse, workspace): 0, or with workspace None the bytes
 * that it has to have (nothing launched) */
ENTRY(attention_call)
{
    amp_attention_args P;
    DLTensor q, kc, vc, out, t;
    cudaStream_t st;
    int dev;
    long window, sinks, bytes;
    double scale;
    if (!count("attention_call", n, 12)) return NULL;
    memset(&P, 0, sizeof P);
    if (!tc_get(a[0], &q, -1) || !tc_rows(&q) || !tc_half(&q, &P.bf16) || q.shape[0] < 1 || q.shape[1] < 1) Py_RETURN_NONE;
    dev = q.device.device_id;
    if (!tc_get(a[1], &kc, dev) || !tc_same(&kc, &q) || kc.ndim != 4 || kc.shape[2] < 1 || !tc_fits(kc.shape[2]) || !tc_cache(&kc, kc.shape[2], q.shape[2])) Py_RETURN_NONE;
    if (!tc_get(a[2], &vc, dev) || !tc_same(&vc, &q) || !tc_cache(&vc, kc.shape[2], q.shape[2]) || vc.shape[0] != kc.shape[0] || vc.shape[1] != kc.shape[1]) Py_RETURN_NONE;
    if (!tc_sequences(a[4], a[5], q.shape[0], dev, &P.pos, &P.cu, &P.seqs, &P.pos64)) Py_RETURN_NONE;
    if (!tc_table(a[3], P.seqs, kc.shape[1], dev, &P.table, &P.table_row, &P.max_pages)) Py_RETURN_NONE;
    if (!tc_get(a[9], &out, dev) || !tc_rows(&out) || !tc_same(&out, &q) || !tc_shape(&out, q.shape[0], q.shape[1], q.shape[2]) || !tc_apart(&out)) Py_RETURN_NONE;
    window = PyLong_AsLong(a[6]);
    sinks = PyLong_AsLong(a[7]);
    scale = PyFloat_AsDouble(a[8]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (window < 0 || sinks < 0 || !(scale - scale == 0.0) || q.shape[1] % kc.shape[2] || tc_ptr(&out) == tc_ptr(&q)) Py_RETURN_NONE;
    if (q.shape[2] != 64 && q.shape[2] != 128 && q.shape[2] != 256) Py_RETURN_NONE;
    P.q = tc_ptr(&q); P.k_cache = tc_ptr(&kc); P.v_cache = tc_ptr(&vc); P.out = tc_ptr(&out);
    P.q_token = tc_stride(&q, 0); P.q_head = tc_stride(&q, 1); P.out_token = tc_stride(&out, 0); P.out_head = tc_stride(&out, 1);
    P.k_page = tc_stride(&kc, 0); P.k_row = tc_stride(&kc, 1); P.k_head = tc_stride(&kc, 2);
    P.v_page = tc_stride(&vc, 0); P.v_row = tc_stride(&vc, 1); P.v_head = tc_stride(&vc, 2);
    P.tokens = (int) q.shape[0]; P.heads = (int) q.shape[1]; P.kv_heads = (int) kc.shape[2]; P.dim = (int) q.shape[2];
    P.pages = (int) kc.shape[0]; P.page_size = (int) kc.shape[1];
    P.window = window < (1 << 30) ? (int) window : 1 << 30; P.sinks = sinks < (1 << 30) ? (int) sinks : 1 << 30;
    P.scale = (float) scale;
    if (a[10] != Py_None)
    {
        if (!tc_get(a[10], &t, dev) || t.ndim != 2 || !tc_is(&t, kDLFloat, 32) || t.shape[0] != q.shape[0] || t.shape[1] != q.shape[1] ||
            !tc_dense(&t, 1) || (t.shape[0] > 1 && t.strides[0] != t.shape[1])) Py_RETURN_NONE;
        P.lse = (float*) tc_ptr(&t);
    }
    if (!tc_stream(dev, &st)) Py_RETURN_NONE;
    bytes = amp_b200_attention_workspace(P.tokens, P.seqs, P.heads, P.kv_heads, P.dim, P.cu != NULL, (long) P.max_pages * P.page_size, P.window, P.sinks);
    if (bytes < 0) Py_RETURN_NONE;
    if (bytes)
    {
        if (a[11] == Py_None) return PyLong_FromLong(bytes);
        if (!tc_get(a[11], &t, dev) || t.ndim != 1 || !tc_dense(&t, 0) || t.dtype.bits != 8 || t.shape[0] < bytes) Py_RETURN_NONE;
        P.workspace = tc_ptr(&t); P.workspace_bytes = (long) t.shape[0];
    }
    TC_RUN(amp_b200_attention(&P, st));
}

#define TC_MAX_PAIRS 64
#define TC_MAX_CACHES 64

/* copy_call(caches, src, dst): lists of tensors and of page numbers, short ones */
ENTRY(copy_call)
{
    DLTensor first, t;
    void* base[TC_MAX_CACHES];
    long layer[TC_MAX_CACHES], page[TC_MAX_CACHES], bytes;
    int src[TC_MAX_PAIRS], dst[TC_MAX_PAIRS], lead = 0;
    cudaStream_t st;
    Py_ssize_t nc, np, i;
    int d;
    if (!count("copy_call", n, 3)) return NULL;
    if (!PyList_CheckExact(a[0]) || !PyList_CheckExact(a[1]) || !PyList_CheckExact(a[2])) Py_RETURN_NONE;
    nc = PyList_GET_SIZE(a[0]); np = PyList_GET_SIZE(a[1]);
    if (nc < 1 || nc > TC_MAX_CACHES || np > TC_MAX_PAIRS || PyList_GET_SIZE(a[2]) != np) Py_RETURN_NONE;
    for (i = 0; i < np; ++i)
    {
        PyObject *x = PyList_GET_ITEM(a[1], i), *y = PyList_GET_ITEM(a[2], i);
        if (!PyLong_CheckExact(x) || !PyLong_CheckExact(y)) Py_RETURN_NONE;
        if (!get_i(x, &src[i]) || !get_i(y, &dst[i])) { PyErr_Clear(); Py_RETURN_NONE; }
    }
    for (i = 0; i < nc; ++i)
    {
        long gap = 1;
        int left;
        if (!tc_get(PyList_GET_ITEM(a[0], i), &t, i ? first.device.device_id : -1)) Py_RETURN_NONE;
        if (i == 0)
        {
            first = t;
            if (t.ndim != 4 && t.ndim != 5) Py_RETURN_NONE;
            lead = t.ndim - 4;
            for (d = 0; d < t.ndim; ++d) if (!tc_fits(t.shape[d]) || t.shape[d] < 1) Py_RETURN_NONE;
        }
        if (t.ndim != first.ndim || !tc_same(&t, &first)) Py_RETURN_NONE;
        for (d = 0; d < t.ndim; ++d) if (t.shape[d] != first.shape[d]) Py_RETURN_NONE;
        /* the three inner dimensions without gaps, in any order */
        for (left = 3; left > 0; )
        {
            int found = 0;
            for (d = lead + 1; d < t.ndim; ++d)
                if (t.shape[d] > 1 && t.strides[d] == gap) { gap *= (long) t.shape[d]; found = 1; break; }
            if (!found) break;
            --left;
        }
        if (gap != t.shape[lead + 1] * t.shape[lead + 2] * t.shape[lead + 3]) Py_RETURN_NONE;
        base[i] = tc_ptr(&t);
        layer[i] = lead ? tc_stride(&t, 0) * (t.dtype.bits / 8) : 0;
        page[i] = tc_stride(&t, lead) * (t.dtype.bits / 8);
    }
    if (first.dtype.bits % 8) Py_RETURN_NONE;
    bytes = (long) (first.shape[lead + 1] * first.shape[lead + 2] * first.shape[lead + 3]) * (first.dtype.bits / 8);
    if (!tc_stream(first.device.device_id, &st)) Py_RETURN_NONE;
    TC_RUN(amp_b200_copy_pages(base, layer, page, (int) nc, lead ? (int) first.shape[0] : 1, (int) first.shape[lead], bytes, src, dst, (int) np, st));
}
#endif
