// adamw_host.cpp -- the per-step host work of AdamW.step() / AdamW8bit.step(),
// of AdamW8bit.moments() and of grad_norm() / clip_grad_norm_() in C++.
//
// A plan is built from the param groups and the state in one call, once every
// parameter with a gradient has its state: one descriptor for each, with all
// but the gradient's address and the scalars filled in.  A step checks that
// nothing the plan relies on has changed (as in smo_host.cpp), fills those in
// and calls smo_adamw_step().  Where a check fails nothing has been modified
// and the caller builds a new plan; where none can be built (a parameter that
// is not contiguous, several devices), the Python path steps.

#include "smo_host.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <unordered_map>
#include <utility>
#include <vector>

#include <ATen/ops/empty.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "smo_b200.h"

namespace smo_host {
namespace {

using AdamwStepFn = int (*)(const smo_adamw_tensor *, int32_t, const float *, float, float *, void *, size_t, void *);
using AdamwAdvanceFn = int (*)(const smo_adamw_schedule *, int32_t, smo_adamw_hyper *, void *);
using AdamwDecodeFn = int (*)(const smo_adamw_tensor *, int32_t, void *);
using GradNormFn = int (*)(const smo_grad *, int32_t, float, float *, void *, size_t, void *);
using WorkspaceFn = size_t (*)(int32_t);

PyObject *s_exp_avg, *s_exp_avg_sq, *s_m_q, *s_m_s, *s_v_q, *s_v_s, *s_master;

constexpr int kMaxKeys = 5;  // state tensors of one parameter

struct AdamEntry {
    PyObject *param = nullptr;  // owned
    PyObject *state = nullptr;  // owned; null: no gradient when the plan was made
    int group = 0;
    int nkeys = 0;
    Py_ssize_t nstate = 0;           // entries of the state
    PyObject *keys[kMaxKeys] = {};   // borrowed (interned)
    PyObject *held[kMaxKeys] = {};   // owned: the state's tensors
    void *held_ptr[kMaxKeys] = {};   // and the addresses the descriptor holds
    void *param_ptr = nullptr;
    std::vector<int64_t> sizes, strides;
    PyObject *step = nullptr;        // owned: the state's step tensor (capturable plans)
    float *step_ptr = nullptr;
    smo_adamw_tensor row;
};

struct AdamGroup {
    PyObject *dict = nullptr;    // owned
    PyObject *params = nullptr;  // owned
    Py_ssize_t n = 0;
};

struct AdamPlan {
    PyObject *groups_list = nullptr;  // owned
    std::vector<AdamGroup> groups;
    std::vector<AdamEntry> entries;
    int device = -1;
    int32_t rows = 0;
    AdamwStepFn step_fn = nullptr;
    AdamwAdvanceFn advance_fn = nullptr;  // capturable: scalars are formed on the device
    unsigned long long generation = 0;
    std::vector<smo_adamw_tensor> table;
    std::vector<smo_adamw_schedule> schedule;
    std::vector<const float *> lr_dev;    // per group
    std::unordered_map<PyObject *, int> coded;  // entries with 8-bit moments, by parameter
    std::vector<long long> next_step;
    std::vector<double> hp_in;

    ~AdamPlan() {
        for (AdamEntry &e : entries) {
            Py_XDECREF(e.param);
            Py_XDECREF(e.state);
            Py_XDECREF(e.step);
            for (PyObject *h : e.held) Py_XDECREF(h);
        }
        for (AdamGroup &g : groups) {
            Py_XDECREF(g.dict);
            Py_XDECREF(g.params);
        }
        Py_XDECREF(groups_list);
    }
};

void plan_free(PyObject *cap) { delete (AdamPlan *)PyCapsule_GetPointer(cap, "smo_adamw_plan"); }

smo_adamw_hyper make_hyper(const double *in, long long step) {
    const double lr = in[0], b1 = in[1], b2 = in[2], eps = in[3], wd = in[4];
    smo_adamw_hyper h;
    h.beta1 = (float)b1;
    h.omb1 = (float)(1.0 - b1);
    h.beta2 = (float)b2;
    h.omb2 = (float)(1.0 - b2);
    h.decay = (float)(1.0 - lr * wd);
    h.step_size = (float)(lr / (1.0 - std::pow(b1, (double)step)));
    h.rsqrt_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(b2, (double)step)));
    h.eps = (float)eps;
    return h;
}

int32_t dtype_code(c10::ScalarType t) {
    switch (t) {
        case c10::ScalarType::Float: return SMO_DTYPE_F32;
        case c10::ScalarType::BFloat16: return SMO_DTYPE_BF16;
        case c10::ScalarType::Half: return SMO_DTYPE_F16;
        default: return -1;
    }
}

// torch refuses to write such a tensor in place: the Python path says so before anything is written
bool not_writable(const at::Tensor &t) { return t.is_inference() && !c10::InferenceMode::is_enabled(); }

// element k of one's memory is element k of the other's (a size of 1 may have any stride)
bool same_layout(const at::Tensor &a, const at::Tensor &b) {
    return a.layout() == c10::kStrided && b.layout() == c10::kStrided && a.device() == b.device() &&
           a.sizes() == b.sizes() && (a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous()));
}

// the state's tensor `key`, or null
PyObject *state_tensor(PyObject *state, PyObject *key) {
    PyObject *t = PyDict_GetItemWithError(state, key);
    return t && THPVariable_Check(t) ? t : nullptr;
}

// codes and scales of n elements: contiguous, of their types, on the device; the block size, or 0
int32_t codes_block(PyObject *const *t, const at::Tensor &p) {
    const at::Tensor &mq = THPVariable_Unpack(t[0]), &ms = THPVariable_Unpack(t[1]);
    const at::Tensor &vq = THPVariable_Unpack(t[2]), &vs = THPVariable_Unpack(t[3]);
    if (mq.scalar_type() != c10::ScalarType::Char || vq.scalar_type() != c10::ScalarType::Byte ||
        ms.scalar_type() != c10::ScalarType::Float || vs.scalar_type() != c10::ScalarType::Float)
        return 0;
    for (int k = 0; k < 4; k++) {
        const at::Tensor &x = THPVariable_Unpack(t[k]);
        if (x.device() != p.device() || x.layout() != c10::kStrided || !x.is_contiguous()) return 0;
    }
    if (mq.dim() != 2 || vq.sizes() != mq.sizes()) return 0;
    const int64_t b = mq.size(1), nb = mq.size(0);
    if ((b != 64 && b != 128 && b != 256) || nb != (p.numel() + b - 1) / b) return 0;
    if (ms.numel() != nb || vs.numel() != nb) return 0;
    return (int32_t)b;
}

// Fills an entry from its parameter, gradient and state; false: not steppable as it is.
bool fill_entry(AdamEntry &e, const at::Tensor &p, const at::Tensor &g) {
    const int32_t dt = dtype_code(p.scalar_type());
    if (dt < 0 || p.layout() != c10::kStrided || !p.is_non_overlapping_and_dense()) return false;
    if (g.scalar_type() != p.scalar_type() || !same_layout(p, g)) return false;
    PyObject *t[kMaxKeys] = {};
    std::memset(&e.row, 0, sizeof(e.row));
    e.row.param = p.data_ptr();
    e.row.n = p.numel();
    e.row.dtype = dt;
    t[0] = state_tensor(e.state, s_exp_avg);
    if (t[0]) {
        t[1] = state_tensor(e.state, s_exp_avg_sq);
        if (!t[1]) return false;
        const at::Tensor &m = THPVariable_Unpack(t[0]), &v = THPVariable_Unpack(t[1]);
        if (m.scalar_type() != c10::ScalarType::Float || v.scalar_type() != c10::ScalarType::Float) return false;
        if (!same_layout(p, m) || !same_layout(p, v)) return false;
        e.row.kind = SMO_ADAMW_F32;
        e.row.exp_avg = (float *)m.data_ptr();
        e.row.exp_avg_sq = (float *)v.data_ptr();
        e.keys[0] = s_exp_avg;
        e.keys[1] = s_exp_avg_sq;
        e.nkeys = 2;
    } else {
        PyObject *const keys[4] = {s_m_q, s_m_s, s_v_q, s_v_s};
        for (int k = 0; k < 4; k++) {
            e.keys[k] = keys[k];
            t[k] = state_tensor(e.state, keys[k]);
            if (!t[k]) return false;
        }
        if (!p.is_contiguous()) return false;  // codes follow the logical order
        e.row.q_block = codes_block(t, p);
        if (!e.row.q_block) return false;
        e.row.kind = SMO_ADAMW_8BIT;
        e.row.m_q = (int8_t *)THPVariable_Unpack(t[0]).data_ptr();
        e.row.m_s = (float *)THPVariable_Unpack(t[1]).data_ptr();
        e.row.v_q = (uint8_t *)THPVariable_Unpack(t[2]).data_ptr();
        e.row.v_s = (float *)THPVariable_Unpack(t[3]).data_ptr();
        e.nkeys = 4;
    }
    if (PyObject *w = state_tensor(e.state, s_master)) {
        const at::Tensor &m = THPVariable_Unpack(w);
        if (dt == SMO_DTYPE_F32 || m.scalar_type() != c10::ScalarType::Float || !same_layout(p, m)) return false;
        e.row.master = (float *)m.data_ptr();
        e.keys[e.nkeys] = s_master;
        t[e.nkeys++] = w;
    }
    for (int k = 0; k < e.nkeys; k++) {
        Py_INCREF(t[k]);
        e.held[k] = t[k];
        e.held_ptr[k] = THPVariable_Unpack(t[k]).data_ptr();
    }
    e.nstate = PyDict_GET_SIZE(e.state);
    e.param_ptr = p.data_ptr();
    e.sizes.assign(p.sizes().begin(), p.sizes().end());
    e.strides.assign(p.strides().begin(), p.strides().end());
    return true;
}

// the state still holds the tensors that the entry's descriptor points into
bool held_unchanged(const AdamEntry &e) {
    for (int q = 0; q < e.nkeys; q++)
        if (PyDict_GetItemWithError(e.state, e.keys[q]) != e.held[q] ||
            THPVariable_Unpack(e.held[q]).data_ptr() != e.held_ptr[q])
            return false;
    return true;
}

bool read_step(PyObject *state, long long *out) {
    PyObject *st = PyDict_GetItemWithError(state, s_step);
    if (!st || !PyLong_CheckExact(st)) return false;
    int overflow = 0;
    const long long s = PyLong_AsLongLongAndOverflow(st, &overflow);
    if (overflow || s < 0 || s == LLONG_MAX) return false;
    *out = s;
    return true;
}

// the state's step as an fp32 tensor of one element on the device, or null
PyObject *step_tensor(PyObject *state, int device) {
    PyObject *o = state_tensor(state, s_step);
    if (!o) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    const bool ok = t.is_cuda() && t.device().index() == device && t.scalar_type() == c10::ScalarType::Float &&
                    t.numel() == 1 && t.layout() == c10::kStrided;
    return ok ? o : nullptr;
}

// read_group() where the learning rate may be an fp32 tensor of one element on the device
bool read_group_capturable(PyObject *g, int device, double *out, const float **lr_dev) {
    PyObject *lr = PyDict_GetItemWithError(g, s_lr);
    *lr_dev = nullptr;
    if (!lr || !THPVariable_Check(lr)) return read_group(g, out);
    const at::Tensor &t = THPVariable_Unpack(lr);
    if (!t.is_cuda() || t.device().index() != device || t.scalar_type() != c10::ScalarType::Float || t.numel() != 1)
        return false;
    PyObject *plain = PyDict_Copy(g), *zero = PyFloat_FromDouble(0.0);
    const bool ok = plain && zero && PyDict_SetItem(plain, s_lr, zero) == 0 && read_group(plain, out);
    Py_XDECREF(plain);
    Py_XDECREF(zero);
    *lr_dev = (const float *)t.data_ptr();
    return ok;
}

// null with no Python error: no plan for these parameters as they are
PyObject *build_plan(PyObject *groups_list, PyObject *state_map, unsigned long long fn, unsigned long long advance_fn) {
    AdamPlan *pl = new AdamPlan();
    PyObject *cap = PyCapsule_New(pl, "smo_adamw_plan", plan_free);
    if (!cap) {
        delete pl;
        return nullptr;
    }
    const auto none = [cap]() -> PyObject * {
        Py_DECREF(cap);
        return nullptr;
    };
    Py_INCREF(groups_list);
    pl->groups_list = groups_list;
    pl->step_fn = (AdamwStepFn)(uintptr_t)fn;
    pl->advance_fn = (AdamwAdvanceFn)(uintptr_t)advance_fn;
    const Py_ssize_t ng = PyList_GET_SIZE(groups_list);
    pl->groups.resize(ng);
    for (Py_ssize_t gi = 0; gi < ng; gi++) {
        AdamGroup &grp = pl->groups[gi];
        grp.dict = PyList_GET_ITEM(groups_list, gi);
        Py_INCREF(grp.dict);
        if (!PyDict_Check(grp.dict)) return none();
        grp.params = PyDict_GetItemWithError(grp.dict, s_params);
        Py_XINCREF(grp.params);
        if (!grp.params || !PyList_CheckExact(grp.params)) return none();
        grp.n = PyList_GET_SIZE(grp.params);
        for (Py_ssize_t j = 0; j < grp.n; j++) {
            PyObject *param = PyList_GET_ITEM(grp.params, j);
            if (!THPVariable_Check(param)) return none();
            pl->entries.emplace_back();
            AdamEntry &e = pl->entries.back();
            Py_INCREF(param);
            e.param = param;
            e.group = (int)gi;
            const at::Tensor &p = THPVariable_Unpack(param);
            const at::Tensor &g = p.grad();
            if (!g.defined()) continue;
            if (!p.is_cuda() || (pl->device >= 0 && p.device().index() != pl->device)) return none();
            pl->device = p.device().index();
            PyObject *state = PyDict_GetItemWithError(state_map, param);
            long long step;
            if (!state || !PyDict_Check(state)) return none();
            Py_INCREF(state);
            e.state = state;
            if (pl->advance_fn) {
                e.step = step_tensor(state, pl->device);
                if (!e.step) return none();
                Py_INCREF(e.step);
                e.step_ptr = (float *)THPVariable_Unpack(e.step).data_ptr();
            } else if (!read_step(state, &step)) {
                return none();
            }
            if (!fill_entry(e, p, g)) return none();
            if (e.row.kind == SMO_ADAMW_8BIT) pl->coded.emplace(param, (int)pl->entries.size() - 1);
            pl->rows++;
        }
    }
    if (pl->device < 0 || PyErr_Occurred()) return none();
    if (g_watcher < 0 || PyDict_Watch(g_watcher, state_map) < 0) return none();
    pl->generation = g_state_generation;
    pl->table.resize(pl->rows);
    if (pl->advance_fn) pl->schedule.resize(pl->rows);
    pl->lr_dev.resize(ng);
    pl->next_step.resize(pl->entries.size());
    pl->hp_in.resize(5 * ng);
    return cap;
}

// -2: a Python error is set; -1: the plan does not apply (nothing modified); 0: stepped; > 0: smo_status
int run_plan(AdamPlan &pl, const float *scale, float max_norm, float *norm_out, void *ws, size_t ws_bytes,
             smo_adamw_hyper *hypers) {
    if (pl.generation != g_state_generation) return -1;
    if (!PyList_CheckExact(pl.groups_list) || PyList_GET_SIZE(pl.groups_list) != (Py_ssize_t)pl.groups.size())
        return -1;
    size_t k = 0;
    for (size_t gi = 0; gi < pl.groups.size(); gi++) {
        const AdamGroup &g = pl.groups[gi];
        if (PyList_GET_ITEM(pl.groups_list, gi) != g.dict) return -1;
        PyObject *ps = PyDict_GetItemWithError(g.dict, s_params);
        if (ps != g.params || PyList_GET_SIZE(ps) != g.n) return -1;
        for (Py_ssize_t j = 0; j < g.n; j++, k++)
            if (PyList_GET_ITEM(ps, j) != pl.entries[k].param) return -1;
        if (pl.advance_fn ? !read_group_capturable(g.dict, pl.device, &pl.hp_in[5 * gi], &pl.lr_dev[gi])
                          : !read_group(g.dict, &pl.hp_in[5 * gi]))
            return -1;
    }
    size_t m = 0;
    int last_group = -1;
    long long last_step = -1;
    smo_adamw_hyper hp{};
    for (size_t i = 0; i < pl.entries.size(); i++) {
        const AdamEntry &e = pl.entries[i];
        const at::Tensor &p = THPVariable_Unpack(e.param);
        const at::Tensor &g = p.grad();
        if (!e.state) {
            if (g.defined()) return -1;
            continue;
        }
        if (!g.defined() || p.data_ptr() != e.param_ptr || not_writable(p)) return -1;
        if (dtype_code(p.scalar_type()) != e.row.dtype || p.device().index() != pl.device) return -1;
        if (p.sizes() != c10::IntArrayRef(e.sizes) || p.strides() != c10::IntArrayRef(e.strides)) return -1;
        if (g.scalar_type() != p.scalar_type() || !same_layout(p, g)) return -1;
        if (!held_unchanged(e)) return -1;
        // a moment or a master copy that came or went makes another kind of entry
        if (PyDict_GET_SIZE(e.state) != e.nstate) return -1;
        smo_adamw_tensor &r = pl.table[m];
        r = e.row;
        r.grad = g.data_ptr();
        if (pl.advance_fn) {
            if (PyDict_GetItemWithError(e.state, s_step) != e.step ||
                THPVariable_Unpack(e.step).data_ptr() != e.step_ptr)
                return -1;
            const double *in = &pl.hp_in[5 * e.group];
            pl.schedule[m] = smo_adamw_schedule{e.step_ptr, pl.lr_dev[e.group], in[0], in[1], in[2], in[3], in[4]};
            r.hp_dev = hypers + m;
        } else {
            long long step;
            if (!read_step(e.state, &step)) return -1;
            pl.next_step[i] = ++step;
            if (e.group != last_group || step != last_step) {
                hp = make_hyper(&pl.hp_in[5 * e.group], step);
                last_group = e.group;
                last_step = step;
            }
            r.hp = hp;
        }
        m++;
    }
    int rc = SMO_OK;
    {
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)pl.device);
        cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)pl.device).stream();
        if (pl.advance_fn) rc = pl.advance_fn(pl.schedule.data(), (int32_t)m, hypers, (void *)stream);
        if (rc != SMO_OK) return rc;
        rc = pl.step_fn(pl.table.data(), (int32_t)m, scale, max_norm, norm_out, ws, ws_bytes, (void *)stream);
    }
    if (rc != SMO_OK) return rc;
    // autograd sees that the parameters were written
    for (const AdamEntry &e : pl.entries)
        if (e.state) THPVariable_Unpack(e.param).unsafeGetTensorImpl()->bump_version();
    if (pl.advance_fn) return SMO_OK;
    for (size_t i = 0; i < pl.entries.size(); i++) {
        if (!pl.entries[i].state) continue;
        PyObject *ns = PyLong_FromLongLong(pl.next_step[i]);
        if (!ns || PyDict_SetItem(pl.entries[i].state, s_step, ns) < 0) {
            Py_XDECREF(ns);
            return -2;
        }
        Py_DECREF(ns);
    }
    return 0;
}

}  // namespace

bool adamw_init() {
    s_exp_avg = PyUnicode_InternFromString("exp_avg");
    s_exp_avg_sq = PyUnicode_InternFromString("exp_avg_sq");
    s_m_q = PyUnicode_InternFromString("m_q");
    s_m_s = PyUnicode_InternFromString("m_s");
    s_v_q = PyUnicode_InternFromString("v_q");
    s_v_s = PyUnicode_InternFromString("v_s");
    s_master = PyUnicode_InternFromString("master");
    return s_exp_avg && s_exp_avg_sq && s_m_q && s_m_s && s_v_q && s_v_s && s_master;
}

// adamw_plan(param_groups, state_mapping, step_fn_addr, advance_fn_addr) -> (capsule, device index, tensors) or
// None; advance_fn_addr is 0 unless the step counts are device tensors
PyObject *adamw_plan(PyObject *, PyObject *args) {
    PyObject *groups_list, *state_map;
    unsigned long long fn, advance_fn;
    if (!PyArg_ParseTuple(args, "O!O!KK", &PyList_Type, &groups_list, &PyDict_Type, &state_map, &fn, &advance_fn))
        return nullptr;
    try {
        PyObject *cap = build_plan(groups_list, state_map, fn, advance_fn);
        if (!cap) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        const AdamPlan *pl = (AdamPlan *)PyCapsule_GetPointer(cap, "smo_adamw_plan");
        return Py_BuildValue("Nii", cap, pl->device, (int)pl->rows);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// adamw_run(capsule, address of the scalars' device memory or 0, grad_scale address or 0, max_norm or 0, norm
// address or 0, workspace address, bytes)
PyObject *adamw_run(PyObject *, PyObject *args) {
    PyObject *cap;
    unsigned long long hypers, scale, norm_out, ws, ws_bytes;
    float max_norm;
    if (!PyArg_ParseTuple(args, "OKKfKKK", &cap, &hypers, &scale, &max_norm, &norm_out, &ws, &ws_bytes)) return nullptr;
    AdamPlan *pl = (AdamPlan *)PyCapsule_GetPointer(cap, "smo_adamw_plan");
    if (!pl) return nullptr;
    try {
        const int rc = run_plan(*pl, (const float *)(uintptr_t)scale, max_norm, (float *)(uintptr_t)norm_out,
                                (void *)(uintptr_t)ws, (size_t)ws_bytes, (smo_adamw_hyper *)(uintptr_t)hypers);
        if (rc == -2) return nullptr;
        PyErr_Clear();
        return PyLong_FromLong(rc);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject *adamw_hyper_bytes(PyObject *, PyObject *args) {
    double in[5];
    long long step;
    if (!PyArg_ParseTuple(args, "dddddL", &in[0], &in[1], &in[2], &in[3], &in[4], &step)) return nullptr;
    const smo_adamw_hyper h = make_hyper(in, step);
    return PyBytes_FromStringAndSize((const char *)&h, sizeof(h));
}

// adamw_moments(state_mapping, [param], [(exp_avg, exp_avg_sq)], decode_fn_addr, plan capsule or None):
// 0, an smo_status, or -1 where a parameter or an output is not as it has to be.  The plan, made of the same
// mapping, saves looking for and checking the states of its parameters.
PyObject *adamw_moments(PyObject *, PyObject *args) {
    PyObject *state_map, *params, *outs, *cap;
    unsigned long long fn;
    if (!PyArg_ParseTuple(args, "O!O!O!KO", &PyDict_Type, &state_map, &PyList_Type, &params, &PyList_Type, &outs, &fn,
                          &cap))
        return nullptr;
    const AdamPlan *pl = nullptr;
    if (cap != Py_None) {
        pl = (AdamPlan *)PyCapsule_GetPointer(cap, "smo_adamw_plan");
        if (!pl) return nullptr;
        if (pl->generation != g_state_generation) pl = nullptr;
    }
    try {
        const Py_ssize_t n = PyList_GET_SIZE(params);
        if (PyList_GET_SIZE(outs) != n) return PyLong_FromLong(-1);
        std::vector<smo_adamw_tensor> table((size_t)n);
        int device = -1;
        PyObject *const keys[4] = {s_m_q, s_m_s, s_v_q, s_v_s};
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject *param = PyList_GET_ITEM(params, i), *pair = PyList_GET_ITEM(outs, i), *t[4];
            bool ok = THPVariable_Check(param) && PyTuple_Check(pair) && PyTuple_GET_SIZE(pair) == 2 &&
                      THPVariable_Check(PyTuple_GET_ITEM(pair, 0)) && THPVariable_Check(PyTuple_GET_ITEM(pair, 1));
            smo_adamw_tensor &r = table[(size_t)i];
            std::memset(&r, 0, sizeof(r));
            if (ok) {
                const at::Tensor &p = THPVariable_Unpack(param);
                const auto known = pl ? pl->coded.find(param) : std::unordered_map<PyObject *, int>::const_iterator();
                const AdamEntry *e = pl && known != pl->coded.end() ? &pl->entries[(size_t)known->second] : nullptr;
                if (e && (!held_unchanged(*e) || p.numel() != e->row.n || p.device().index() != pl->device)) e = nullptr;
                if (e) {
                    r.m_q = e->row.m_q;
                    r.m_s = e->row.m_s;
                    r.v_q = e->row.v_q;
                    r.v_s = e->row.v_s;
                    r.q_block = e->row.q_block;
                } else {
                    PyObject *state = PyDict_GetItemWithError(state_map, param);
                    ok = p.is_cuda() && state && PyDict_Check(state);
                    for (int k = 0; ok && k < 4; k++) {
                        t[k] = state_tensor(state, keys[k]);
                        ok = t[k] != nullptr;
                    }
                    r.q_block = ok ? codes_block(t, p) : 0;
                    ok = ok && r.q_block;
                    if (ok) {
                        r.m_q = (int8_t *)THPVariable_Unpack(t[0]).data_ptr();
                        r.m_s = (float *)THPVariable_Unpack(t[1]).data_ptr();
                        r.v_q = (uint8_t *)THPVariable_Unpack(t[2]).data_ptr();
                        r.v_s = (float *)THPVariable_Unpack(t[3]).data_ptr();
                    }
                }
                ok = ok && (device < 0 || p.device().index() == device);
                if (ok) device = p.device().index();
                for (int k = 0; ok && k < 2; k++) {
                    const at::Tensor &o = THPVariable_Unpack(PyTuple_GET_ITEM(pair, k));
                    ok = !not_writable(o) && o.scalar_type() == c10::ScalarType::Float && o.device() == p.device() &&
                         o.layout() == c10::kStrided && o.sizes() == p.sizes() && o.is_contiguous();
                    (k ? r.exp_avg_sq : r.exp_avg) = ok ? (float *)o.data_ptr() : nullptr;
                }
                r.n = p.numel();
                r.kind = SMO_ADAMW_8BIT;
            }
            if (!ok) {
                PyErr_Clear();
                return PyLong_FromLong(-1);
            }
        }
        if (n == 0) return PyLong_FromLong(0);
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
        cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        const int rc = ((AdamwDecodeFn)(uintptr_t)fn)(table.data(), (int32_t)n, (void *)stream);
        if (rc == SMO_OK)
            for (Py_ssize_t i = 0; i < n; i++)
                for (int k = 0; k < 2; k++)
                    THPVariable_Unpack(PyTuple_GET_ITEM(PyList_GET_ITEM(outs, i), k)).unsafeGetTensorImpl()->bump_version();
        return PyLong_FromLong(rc);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// grad_norm([parameter], max_norm, norm_fn_addr, workspace_fn_addr) -> (status, norm tensor), or None where a
// gradient is not on the first one's CUDA device, of a known type and one span of memory, is there twice, shares
// elements with another that would both be scaled or must not be written, or there is none
PyObject *grad_norm(PyObject *, PyObject *args) {
    PyObject *list;
    float max_norm;
    unsigned long long fn, ws_fn;
    if (!PyArg_ParseTuple(args, "O!fKK", &PyList_Type, &list, &max_norm, &fn, &ws_fn)) return nullptr;
    try {
        const Py_ssize_t n = PyList_GET_SIZE(list);
        std::vector<smo_grad> table;
        table.reserve((size_t)n);
        int device = -1;
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject *o = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(o)) Py_RETURN_NONE;
            const at::Tensor &g = THPVariable_Unpack(o).grad();
            if (!g.defined()) continue;
            const int32_t dt = dtype_code(g.scalar_type());
            if (dt < 0 || !g.is_cuda() || g.layout() != c10::kStrided || !g.is_non_overlapping_and_dense())
                Py_RETURN_NONE;
            if (max_norm > 0.0f && not_writable(g)) Py_RETURN_NONE;
            if (device >= 0 && g.device().index() != device) Py_RETURN_NONE;
            device = g.device().index();
            table.push_back(smo_grad{g.data_ptr(), g.numel(), dt, 0});
        }
        if (device < 0) Py_RETURN_NONE;
        // a gradient given twice (one address) would be counted twice, and an element that two gradients share
        // scaled by two threads: runs of ascending spans first, mostly a few that are apart
        const auto collide = [&](bool whole_runs) {
            std::vector<std::pair<uintptr_t, uintptr_t>> spans;
            for (const smo_grad &g : table) {
                if (!g.n) continue;
                const uintptr_t a = (uintptr_t)g.grad, bytes = (uintptr_t)g.n * (g.dtype == SMO_DTYPE_F32 ? 4 : 2);
                const uintptr_t end = max_norm > 0.0f ? a + bytes : a + 1;
                if (whole_runs && !spans.empty() && a >= spans.back().second) spans.back().second = end;
                else spans.emplace_back(a, end);
            }
            std::sort(spans.begin(), spans.end());
            for (size_t i = 1; i < spans.size(); i++)
                if (spans[i].first < spans[i - 1].second) return true;
            return false;
        };
        if (collide(true) && collide(false)) Py_RETURN_NONE;
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
        const size_t bytes = ((WorkspaceFn)(uintptr_t)ws_fn)((int32_t)table.size());
        const auto on = at::TensorOptions().device(c10::Device(c10::kCUDA, (c10::DeviceIndex)device));
        at::Tensor out = at::empty({}, on.dtype(c10::ScalarType::Float));
        at::Tensor ws = at::empty({(int64_t)bytes}, on.dtype(c10::ScalarType::Byte));
        cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        const int rc = ((GradNormFn)(uintptr_t)fn)(table.data(), (int32_t)table.size(), max_norm, (float *)out.data_ptr(),
                                                   ws.data_ptr(), bytes, (void *)stream);
        if (rc == SMO_OK && max_norm > 0.0f)
            for (Py_ssize_t i = 0; i < n; i++) {
                const at::Tensor &g = THPVariable_Unpack(PyList_GET_ITEM(list, i)).grad();
                if (g.defined()) g.unsafeGetTensorImpl()->bump_version();
            }
        return Py_BuildValue("iN", rc, THPVariable_Wrap(out));
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

}  // namespace smo_host
