"""Which tests are skipped where the reference can neither be built nor is: none where there is a checkout, or what they
need has been built."""
import os
import re

import pytest

import conftest


@pytest.mark.parametrize("checkout", [False, True])
@pytest.mark.parametrize("oracle,adapter", [(False, False), (True, False), (False, True), (True, True)])
def test_only_what_is_missing_is_skipped(tmp_path, monkeypatch, checkout, oracle, adapter):
    for there, path in ((oracle, "oracle/_ref/libqwen_ref_avx2.so"), (adapter, "qwen3-tts_b200/lib/libqwen_tts_cuda_b200.so")):
        (tmp_path / path).parent.mkdir(parents=True)
        if there:
            (tmp_path / path).touch()
    monkeypatch.setattr(conftest, "ROOT", str(tmp_path))
    monkeypatch.setattr(conftest, "reference_checkout", lambda: "somewhere" if checkout else None)
    want = set() if checkout else {n for n, there in ((conftest.ORACLE, oracle), (conftest.ADAPTER, adapter)) if not there}
    assert set(conftest.reference_missing()) == want


def test_the_names_are_those_of_tests():
    here = os.path.dirname(os.path.abspath(__file__))
    for name, tests in conftest.NEEDS.items():
        with open(os.path.join(here, name)) as f:
            have = set(re.findall(r"^def (test_\w+)", f.read(), re.M))
        assert set(tests) <= have, set(tests) - have
