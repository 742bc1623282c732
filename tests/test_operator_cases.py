"""CPU: the Python package and the operator cases as a program finds them whose working folder is the root of a checkout, with
nothing else on its path."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fresh(code):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout.strip()


def test_the_package_is_found_from_the_root():
    """`import ltq` gives the package itself, its modules included, and only one of it."""
    got = fresh("import sys, ltq, ltq.cache; print(ltq.__file__); print(sys.modules['ltq'] is ltq, ltq.cache.KVCache is ltq.KVCache)")
    assert got.splitlines() == [os.path.join(ROOT, "light-tensor_b200", "python", "ltq", "__init__.py"), "True True"]


@pytest.mark.parametrize("op", ["tokens", "linear", "append", "attention"])
def test_a_case_of_any_operator_may_be_the_first(op):
    """The library's call is reached (and refuses: there is no GPU tensor) whichever operator a process begins with."""
    setup = {"tokens": "state = dict(x=torch.zeros(2, 8))",
             "linear": "import ltq; state = dict(layer=object.__new__(ltq.FullyConnected_t), x=torch.zeros(2, 8))",
             "append": "import ltq; state = dict(cache=object.__new__(ltq.KVCache), new_k=None, new_v=None, table=None, lengths=None, offsets=None, max_new=1)",
             "attention": "import ltq; state = dict(cache=object.__new__(ltq.KVCache), q=None, table=None, lengths=None, offsets=None, max_new=1)"}[op]
    got = fresh(f"""
import importlib.util, torch
spec = importlib.util.spec_from_file_location("cases", "perf/operators.py")
m = importlib.util.module_from_spec(spec)
spec.loader.exec_module(m)
m.own = True
{setup}
state["case"] = dict(op={op!r})
try:
    m.run(state)
except (ValueError, AttributeError) as e:   # (the objects are empty shells)
    print(type(e).__name__)
""")
    assert got == ("ValueError" if op == "tokens" else "AttributeError")
