"""The host side of the operators for many continuations, on a HIP runtime
that runs no kernels (host_hip.cpp): which stream they launch on while a state
captures its decode step, which device is current afterwards, what is waited
for when a launch fails. Each test is a process of its own."""
import os
import subprocess
import sys
import textwrap

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "aot-llm_amd")

COMMON = """
import ctypes as C, sys, threading
import numpy as np
hip = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
for f in ("hh_launched", "hh_foreign", "hh_queued"):
    getattr(hip, f).restype = C.c_long
hip.hh_queued.argtypes = [C.c_void_p]
sys.path.insert(0, sys.argv[2])
import aotk
lib = aotk.abi.load()

mem = np.zeros(1 << 16, np.float32)  # the device's memory is the host's here
P = mem.ctypes.data
OUT = P + (1 << 17)
lens = np.array([3, 2], np.uint32)
table = aotk.logits_rules_table([{}, {}])[0]
calls = {
    "sinks": lambda: lib.aotk_attention_sinks(OUT, P, P + 4096, P + 8192, 0, 1, 1, 64, 4, 0, 3, 1, 0, 0),
    "shared": lambda: lib.aotk_attention_shared(OUT, P, P + 4096, P + 8192, P + 16384, P + 32768, 0, 1, 1, 64, 4, 4, 4, 0, 2,
                                                lens.ctypes.data, None),
    "rules": lambda: lib.aotk_logits_rules(OUT, P, 0, 2, 64, 64, table.ctypes.data, None, 0, None, None, 0, None, 0, None),
}
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("hip") / "libhost_hip.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-pthread", os.path.join(HERE, "host_hip.cpp"), "-o", so],
                   check=True)
    return so


def run(stand_in, body, *args):
    p = subprocess.run([sys.executable, "-c", COMMON + textwrap.dedent(body), stand_in, PKG, *args], capture_output=True, text=True,
                       timeout=300)
    assert p.returncode == 0, p.stdout + p.stderr


@pytest.mark.parametrize("how", ["greedy", "sampled"])
@pytest.mark.parametrize("order", ["capture first", "call first"])
def test_a_state_that_captures_its_decode_step_beside_the_calls(stand_in, how, order):
    """The state's capture takes no launch of another thread's call, and the
    call is not refused for it; both orders of the two."""
    run(stand_in, """
        how, order = sys.argv[3:]
        aotk.init(0)
        model = aotk.Model(aotk.configs.build("tiny-q4km"), seed=3)
        sampler = aotk.Sampler(temperature=1.0, top_k=4)
        for name, call in calls.items():
            failed, rc = [], []

            def generate():
                try:
                    if how == "greedy":
                        aotk.State(model, 32, 8).generate(0, 4)
                    else:
                        aotk.State(model, 32, 8).generate_sampled(sampler, 0, 4, [])
                except aotk.AotkError as e:
                    failed.append(str(e))

            def operator():
                rc.append((call(), lib.aotk_last_error()))

            a, b = threading.Thread(target=generate), threading.Thread(target=operator)
            hip.hh_arm(0)
            if order == "capture first":
                a.start()
                assert hip.hh_reached(0, 10000)
                b.start()
                b.join(10)
            else:
                hip.hh_arm(1)
                b.start()
                assert hip.hh_reached(1, 10000)
                a.start()
                hip.hh_reached(0, 2000)  # unless the state waits for the call
                hip.hh_open(1)
                b.join(10)
            hip.hh_open(0)
            a.join(20)
            b.join(20)
            assert hip.hh_foreign() == 0, (name, "launches of the call are in the state's graph")
            assert rc and rc[0][0] == 0, (name, rc)
            assert not failed, (name, failed)
    """, how, order)


def test_a_capture_from_a_thread_with_another_device_current(stand_in):
    """The step is captured on the library's device; the thread keeps its own."""
    run(stand_in, """
        hip.hh_devices(3)
        aotk.init(2)
        model = aotk.Model(aotk.configs.build("tiny-q4km"), seed=3)
        now = []

        def generate():
            hip.hipSetDevice(1)
            aotk.State(model, 32, 8).generate(0, 4)
            d = C.c_int()
            hip.hipGetDevice(C.byref(d))
            now.append(d.value)

        t = threading.Thread(target=generate)
        t.start()
        t.join()
        assert hip.hh_captured_on() == 2 and now == [1], (hip.hh_captured_on(), now)
    """)


@pytest.mark.parametrize("name", ["sinks", "shared", "rules"])
def test_the_callers_device_is_given_back_by_the_librarys_first_call(stand_in, name):
    """That call initialises the library, on device 0."""
    run(stand_in, """
        hip.hh_devices(3)
        hip.hipSetDevice(1)
        now = C.c_int()
        for turn in range(2):
            assert calls[sys.argv[3]]() == 0, lib.aotk_last_error()
            hip.hipGetDevice(C.byref(now))
            assert now.value == 1, (turn, now.value)
    """, name)


@pytest.mark.parametrize("name", ["sinks", "shared", "rules"])
def test_an_earlier_error_of_the_thread_is_not_the_calls(stand_in, name):
    run(stand_in, """
        assert calls[sys.argv[3]]() == 0
        hip.hh_set_last_error(2)
        assert calls[sys.argv[3]]() == 0, lib.aotk_last_error()
    """, name)


def test_a_launch_that_fails_is_reported_after_the_others_have_ended(stand_in):
    """Of a call of several launches each one fails once: the call says so, and
    nothing of it is left on the stream when it returns."""
    run(stand_in, """
        aotk.init(0)
        stream = aotk.stream()
        many = np.ones(130, np.uint32)
        rules = aotk.logits_rules_table([{}] * 65540)[0]
        big = np.zeros(65540 * 4, np.float32)
        several = {
            "sinks": lambda: lib.aotk_attention_sinks(OUT, P, P + 4096, P + 8192, 0, 1, 1, 64, 200, 0, 199, 1, 0, 0),
            "shared": lambda: lib.aotk_attention_shared(OUT, P, P + 40960, P + 43008, P + 45056, P + 78848, 0, 1, 1, 64, 4, 4, 1, 0,
                                                        130, many.ctypes.data, None),
            "rules": lambda: lib.aotk_logits_rules(big.ctypes.data, big.ctypes.data, 0, 65540, 4, 4, rules.ctypes.data, None, 0, None,
                                                   None, 0, None, 0, None),
        }
        for name, call in several.items():
            before = hip.hh_launched()
            assert call() == 0, (name, lib.aotk_last_error())
            n = hip.hh_launched() - before
            assert n > 1, (name, n)
            for i in range(n):
                hip.hh_fail_launch(i + 1)
                assert call() == -1, (name, i)
                assert b"an error of the stand-in" in lib.aotk_last_error()
                assert hip.hh_queued(stream) == 0, (name, i, "launches that nothing has waited for")
            assert call() == 0, (name, lib.aotk_last_error())
    """)


def test_a_states_mask_beside_a_rule_that_names_one(stand_in):
    """apply_rules takes the mask as its argument: a rule of a batch that says
    otherwise is refused, not followed."""
    run(stand_in, """
        spec = aotk.configs.build("tiny-q4km")
        st = aotk.State(aotk.Model(spec, seed=3), 32, 8)
        mask = aotk.allowed_mask([3], spec.d["vocab"])
        for rule, m in (({}, None), ({}, mask), ({"mask": 0}, mask), ({"mask": -1}, None)):
            st.apply_rules(rule, m)
        for rule, m in (({"mask": -1}, mask), ({"mask": 0}, None), ({"mask": 2}, mask)):
            try:
                st.apply_rules(rule, m)
            except ValueError as e:
                assert "mask" in str(e)
            else:
                raise AssertionError((rule, m is not None))
        try:
            st.apply_rules({}, np.stack([mask, mask]))
        except ValueError as e:
            assert "one row" in str(e)
        else:
            raise AssertionError("two masks")
    """)
