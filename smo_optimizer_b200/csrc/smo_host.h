// smo_host.h -- what the two source files of the _smo_host extension share.
#pragma once

#include <Python.h>

namespace smo_host {

// interned names of param-group and state entries
extern PyObject *s_params, *s_step, *s_lr, *s_betas, *s_eps, *s_weight_decay;

// dict watcher (negative: none was free) and the count of changes it has seen
// to any watched optimizer state mapping
extern int g_watcher;
extern unsigned long long g_state_generation;

// a group's lr, beta1, beta2, eps and weight_decay as doubles (false: one is no plain number)
bool read_group(PyObject *group, double *out);

// adamw_host.cpp: methods of the module
PyObject *adamw_plan(PyObject *, PyObject *args);
PyObject *adamw_run(PyObject *, PyObject *args);
PyObject *adamw_hyper_bytes(PyObject *, PyObject *args);
PyObject *adamw_moments(PyObject *, PyObject *args);
PyObject *grad_norm(PyObject *, PyObject *args);
bool adamw_init();  // interns its names

}  // namespace smo_host
