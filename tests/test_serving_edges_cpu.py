"""The serving operators at their edges, as far as no GPU is needed."""
import os
import random
import subprocess

import torch

from mlir_edsl import _native, serving

INVALID = 1


def test_expire_limits():
    L = _native.lib()
    assert L.b200_debug_w4_expire(-1) == INVALID
    assert "negative" in L.b200_last_error().decode()
    assert L.b200_debug_w4_expire(0) == 0


def test_overlap_of_rows():
    """Against the sets of bytes, over rows of one buffer and several pitches."""
    overlap = serving._calls.overlap_of
    rng = random.Random(1)
    buf = torch.zeros(200, dtype=torch.uint8)
    found = [0, 0]
    for _ in range(4000):
        views, taken = [], []
        for _ in range(2):
            ld, m = rng.choice([5, 8, 8, 8, 13]), rng.randint(0, 5)
            n, start = rng.randint(0, ld), rng.randint(0, 60)
            views.append(buf.as_strided((m, n), (ld, 1), start))
            taken.append({start + i * (ld if m > 1 else n) + k for i in range(m) for k in range(n)})
        want = bool(taken[0] & taken[1])
        found[want] += 1
        assert overlap(*views) == want, (views[0].shape, views[0].stride(), views[1].shape)
    assert min(found) > 500
    cols = torch.zeros(6, 32)
    assert not overlap(cols[:, :16], cols[:, 16:]) and not overlap(cols[:3], cols[3:])
    assert not overlap(cols[:, 4:8], cols[:, 8:32]) and overlap(cols[:, 4:9], cols[:, 8:32])
    assert overlap(cols[:, 30:], cols.view(3, 64)[:, 62:])
    assert not overlap(cols[:, 30:], cols.view(3, 64)[:, :30])


def _run_cpp(tmp_path, body):
    """Compiles and runs a program around csrc/device_facts.h; its main is `body`."""
    csrc = os.path.join(os.path.dirname(_native.__file__), "..", "csrc")
    src, exe = tmp_path / "facts.cpp", tmp_path / "facts"
    src.write_text('#include "device_facts.h"\n#include <atomic>\n#include <cassert>\n#include <thread>\n'
                   "#include <vector>\nint main() {\n" + body + "\nreturn 0;\n}\n")
    subprocess.run(["g++", "-std=c++17", "-UNDEBUG", "-I", csrc, str(src), "-o", str(exe),
                    "-lpthread"], check=True)
    subprocess.run([str(exe)], check=True, timeout=60)


def test_a_failing_query_leaves_no_error_behind(tmp_path):
    _run_cpp(tmp_path, """
      int errors = 0;  // what the next check would find
      auto forget = [&] { errors = 0; };
      auto fails = [&](int* n) { *n = 7; ++errors; return false; };
      assert(b200::ask_or(3, fails, forget) == 3 && errors == 0);
      auto gives = [](int value) { return [=](int* n) { *n = value; return true; }; };
      errors = 5;  // an error that was there before is the caller's
      assert(b200::ask_or(3, gives(4), forget) == 4 && errors == 5);
      assert(b200::ask_or(3, gives(0), forget) == 3 && errors == 5);""")


def test_queries_go_through_it():
    """No occupancy query but those that ask_or makes."""
    csrc = os.path.join(os.path.dirname(_native.__file__), "..", "csrc")
    for name in os.listdir(csrc):
        text = open(os.path.join(csrc, name)).read()
        for part in text.split("cudaOccupancy")[:-1]:
            assert "ask_or(" in part[-200:], name


def test_values_for_each_device(tmp_path):
    _run_cpp(tmp_path, """
      static b200::PerDevice<int> values;
      std::atomic<int> made{0};
      auto of = [&](int device) {
        return values.of(device, [&] { ++made; return 10 * device + 1; });
      };
      std::vector<std::thread> threads;
      for (int t = 0; t < 8; ++t)
        threads.emplace_back([&] { for (int d = 0; d < 64; ++d) assert(of(d) == 10 * d + 1); });
      for (auto& t : threads) t.join();
      assert(made == 64);
      assert(of(64) == 641 && of(64) == 641 && made == 66);  // past the table: asked each time
      assert(of(-1) == -9);""")


def test_nothing_about_one_device_is_kept_for_all():
    """What is kept from a query is kept for its device."""
    csrc = os.path.join(os.path.dirname(_native.__file__), "..", "csrc")
    for name in ("rms_norm.cu", "dense_w4.cu", "dense_w4_tc.cu", "token_logprobs.cu"):
        text = open(os.path.join(csrc, name)).read()
        assert "static const " not in text, name
