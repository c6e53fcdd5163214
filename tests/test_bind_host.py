"""The compiled callers (csrc/bind.c) without a GPU: built against a stand-in for the library whose launches do not return until
another Python thread lets them, with tensors that only claim to be on a device."""
import ctypes as C
import importlib.util
import os
import subprocess
import sysconfig
import threading
import time

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "berth_b200", "csrc")

STUB = r"""
#include <stdatomic.h>
#include <unistd.h>
#include "berth_b200.h"
static atomic_int inside, let;
int stub_inside(void) { return inside; }
void stub_let(int on) { let = on; }
static int wait_for_the_other(void)
{
    ++inside;
    for (int i = 0; i < 10000; ++i) {
        if (let) { --inside; return let > 0 ? 0 : -1; }
        usleep(1000);
    }
    --inside;
    return -1;   /* nobody could: the caller kept the interpreter to itself */
}
int berth_device_current(void) { return 3; }
const char* berth_ops_last_error(void) { return "not let"; }
const char* berth_moe_last_error(void) { return "not let"; }
int berth_ops_rope(const berth_rope_rows* q, const berth_rope_rows* k, const int32_t* positions, const double* inv_freq, int n_tokens, int head_dim,
                   int rot_dim, int interleaved, float attention_factor, float norm_epsilon, float norm_bias, int fp32, void* stream)
{ return wait_for_the_other(); }
int berth_ops_logprobs(const void* logits, int logits_fp32, int64_t row_stride, const int32_t* tokens, float inv_temp, float* logprob, int32_t* rank,
                       float* entropy, int32_t* top_idx, float* top_logprob, int top_n, int rows, int vocab, void* stream)
{ return wait_for_the_other(); }
int berth_moe_route(const void* logits, int logits_fp32, int64_t row_stride, const float* selection_bias, int32_t* topk_idx, float* topk_w, int T,
                    int n_experts, int top_k, int score, int n_group, int topk_group, int group_score, int renormalize, float scale, void* stream)
{ return wait_for_the_other(); }
"""


class DlTensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("device_type", C.c_int32), ("device_id", C.c_int32), ("ndim", C.c_int32), ("code", C.c_uint8), ("bits", C.c_uint8),
                ("lanes", C.c_uint16), ("shape", C.POINTER(C.c_int64)), ("strides", C.POINTER(C.c_int64)), ("byte_offset", C.c_uint64)]


class DlExchange(C.Structure):
    _fields_ = [("major", C.c_uint32), ("minor", C.c_uint32)] + [(n, C.c_void_p) for n in (
        "previous", "allocate", "managed_from_object", "managed_to_object", "tensor_from_object", "current_stream")]


class Claims:
    """What the callers read of a tensor: on device 3, contiguous, at an address that nothing reads."""

    def __init__(self, kind, *shape):
        self.shape = (C.c_int64 * 3)(*shape)
        strides = [1]
        for n in reversed(shape[1:]):
            strides.insert(0, strides[0] * n)
        self.strides = (C.c_int64 * 3)(*strides)
        self.ndim, (self.code, self.bits) = len(shape), kind


HALF, FLOAT, DOUBLE, INT = (2, 16), (2, 32), (2, 64), (0, 32)


@C.PYFUNCTYPE(C.c_int, C.py_object, C.POINTER(DlTensor))
def _read(o, out):
    t = out.contents
    t.data, t.device_type, t.device_id, t.ndim, t.code, t.bits, t.lanes, t.byte_offset = 4096, 2, 3, o.ndim, o.code, o.bits, 1, 0
    t.shape, t.strides = C.cast(o.shape, C.POINTER(C.c_int64)), C.cast(o.strides, C.POINTER(C.c_int64))
    return 0


_exchange = DlExchange(1, 0, None, None, None, None, C.cast(_read, C.c_void_p), None)
_capsule_new = C.pythonapi.PyCapsule_New
_capsule_new.restype, _capsule_new.argtypes = C.py_object, [C.c_void_p, C.c_char_p, C.c_void_p]
_name = C.create_string_buffer(b"dlpack_exchange_api")   # the capsule keeps its address
Claims.__dlpack_c_exchange_api__ = _capsule_new(C.addressof(_exchange), C.cast(_name, C.c_char_p), None)


class Refused(RuntimeError):
    pass


@pytest.fixture(scope="module")
def stubbed(tmp_path_factory):
    """(the callers, the stand-in)"""
    d = tmp_path_factory.mktemp("bind")
    (d / "stub.c").write_text(STUB)
    so = str(d / "_bind.so")
    subprocess.run(["gcc", "-O1", "-std=c11", "-D_DEFAULT_SOURCE", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-I" + sysconfig.get_paths()["include"],
                    "-I" + os.path.join(CSRC, "..", "..", "include"), os.path.join(CSRC, "bind.c"), str(d / "stub.c"), "-o", so], check=True)
    spec = importlib.util.spec_from_file_location("_bind", so)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.init(Refused, Claims)
    return module, C.CDLL(so)


def _calls(module):
    return {
        "rope": lambda: module.rope(Claims(HALF, 3, 4, 64), None, Claims(INT, 3), Claims(DOUBLE, 32), Claims(HALF, 3, 4, 64), None, False, 1.0, None, None,
                                    1e-6, 0.0, None),
        "logprobs": lambda: module.logprobs(Claims(FLOAT, 3, 50), None, None, None, Claims(FLOAT, 3), None, None, None, 1.0, None),
        "route": lambda: module.route(Claims(FLOAT, 3, 64), None, Claims(INT, 3, 4), Claims(FLOAT, 3, 4), 4, 0, 1, 1, 0, True, 1.0, None)}


def _start(stubbed, name, threads):
    """The threads' results, once so many launches were under way at once and were let go with `verdict`."""
    module, stub = stubbed

    def run(verdict):
        stub.stub_let(0)
        said = []

        def caller():
            try:
                said.append(_calls(module)[name]())
            except Refused as e:
                said.append(str(e))
        ts = [threading.Thread(target=caller) for _ in range(threads)]
        for t in ts:
            t.start()
        while stub.stub_inside() < threads and any(t.is_alive() for t in ts):
            time.sleep(0.001)
        together = stub.stub_inside()
        stub.stub_let(verdict)
        for t in ts:
            t.join()
        return said, together
    return run


@pytest.mark.parametrize("name", ["rope", "logprobs", "route"])
def test_a_launch_that_blocks_leaves_other_threads_running(stubbed, name):
    """The launch of one thread returns only after another one has run Python code."""
    said, together = _start(stubbed, name, 1)(1)
    assert said == [None] and together == 1


@pytest.mark.parametrize("name", ["rope", "logprobs", "route"])
def test_two_threads_launch_side_by_side(stubbed, name):
    """Two threads in the library at once; both end with what the call returned, an error among it."""
    run = _start(stubbed, name, 2)
    assert run(1) == ([None, None], 2)
    assert run(-1) == (["not let", "not let"], 2)


def test_a_torch_without_the_exchange_interface_is_named(stubbed, monkeypatch):
    """init() and the package's bind() say which interface is missing, in which torch, and which torch has it; init() keeps what it has."""
    module, _ = stubbed

    class Bare:
        pass
    with pytest.raises(ImportError, match="__dlpack_c_exchange_api__.*torch 2.11"):
        module.init(Refused, Bare)
    old = DlExchange(0, 9, None, None, None, None, C.cast(_read, C.c_void_p), None)

    class Other:
        __dlpack_c_exchange_api__ = _capsule_new(C.addressof(old), C.cast(_name, C.c_char_p), None)
    with pytest.raises(ImportError, match="DLPack 0.9.*torch 2.11"):
        module.init(Refused, Other)
    with pytest.raises(Refused, match="must be a torch tensor"):      # still those of the first init
        module.route(Bare(), *[None] * 11)

    import torch
    from berth_b200 import _lib
    monkeypatch.setattr(_lib, "_bind", None)
    monkeypatch.setattr(torch, "Tensor", Bare)
    with pytest.raises(ImportError, match="__dlpack_c_exchange_api__"):
        _lib.bind()
    assert _lib._bind is None
