"""Shared test setup.

- registers the `gpu` marker (tests that need a B200 and the built CUDA engine);
- puts the engine's Python bindings (qwen3-tts_b200/) and the parity oracle
  (oracle/, test infrastructure) on sys.path;
- selects the reference's f32-activation kernels for the oracle process
  (QWEN_NO_BF16DOT / QWEN_NO_VNNI / QWEN_NO_SDOT = 1, the semantics the
  reference's own `make test-selftest` fallback run uses, Makefile:756-761);
- selects the reference's sequential code-predictor prefill
  (QWEN_CP_PREFILL2 = 0): positions 0 and 1 one at a time, as its GPU path
  runs them (qwen_cuda_cp_step per position).  Its fused two-position variant
  caches its mode per thread on first use (qwen_tts_code_predictor.c:784), so
  a process that runs a quantized code predictor and then a bf16 one takes the
  quantized branch on bf16 weights and crashes;
- skips the tests that compare with the compiled reference where there is
  neither a checkout of it to build from nor what was built from one.
"""
import glob
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "qwen3-tts_b200"))
sys.path.insert(0, os.path.join(ROOT, "oracle"))
sys.path.insert(0, ROOT)
from __graft_entry__ import _ref_checkout as reference_checkout  # noqa: E402
for _k, _v in {"QWEN_NO_BF16DOT": "1", "QWEN_NO_VNNI": "1", "QWEN_NO_SDOT": "1", "QWEN_CP_PREFILL2": "0"}.items():
    os.environ.setdefault(_k, _v)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 GPU and the built sm_100a engine")
    config.addinivalue_line("markers", "slow: full-size model cases (tens of seconds)")


# What the tests need that is built from a reference checkout: the compiled
# reference (oracle/_ref), the library compiled against its headers (adapter).
ORACLE, ADAPTER = "oracle", "adapter"
NEEDS = {
    "test_abi.py": {
        "test_engine_library_exports_everything_declared": (ADAPTER,),
        "test_dropin_surface_matches_reference_names": (ADAPTER,)},
    "test_oracle_pin.py": {n: (ORACLE,) for n in (
        "test_matvec_bf16_int8_q4_0_against_reference", "test_int8_encoder_bit_exact", "test_q4_0_encoder_bit_exact",
        "test_attention_norms_swiglu_against_reference", "test_talker_steps_match_reference",
        "test_cp_predict_matches_reference", "test_sampler_matches_reference")},
    "test_gpu_dispatch.py": {"test_default_dispatch_gap": (ORACLE,)},
    "test_gpu_dropin.py": {"test_batched_dropin_entry_points": (ORACLE, ADAPTER)},
    "test_gpu_fullsize.py": {n: (ORACLE,) for n in (
        "test_c2_06b_int8_64_frames_match_reference", "test_c3_17b_q4_0_talker_matches_reference",
        "test_c5_17b_cp_with_mtp_codes_identical")},
    "test_gpu_kernels.py": {n: (ORACLE,) for n in (
        "test_kv_append_bit_exact_vs_reference", "test_codec_sampler_matches_reference")},
    "test_gpu_model.py": {**{n: (ORACLE,) for n in (
        "test_talker_steps_match_reference", "test_cp_frame_codes_match_reference", "test_prefill_matches_reference_prefill",
        "test_decode_frames_match_reference_loop", "test_generation_rules_eos_and_repetition_match_reference",
        "test_sampling_frames_match_reference", "test_06b_bf16_greedy_256_steps_identical")},
        "test_dropin_reference_delegates_to_engine": (ORACLE, ADAPTER)},
    "test_gpu_refcuda.py": {n: (ORACLE,) for n in (
        "test_reference_cuda_path_agrees_on_tiny_model", "test_reference_cuda_path_timed_against_engine")},
}


def reference_missing():
    """What is neither built nor can be: {} wherever there is a reference checkout."""
    if reference_checkout():
        return {}
    built = {ORACLE: glob.glob(os.path.join(ROOT, "oracle", "_ref", "libqwen_ref_*.so")),
             ADAPTER: glob.glob(os.path.join(ROOT, "qwen3-tts_b200", "lib", "libqwen_tts_cuda_b200.so"))}
    said = {ORACLE: "the compiled reference (oracle/_ref)", ADAPTER: "libqwen_tts_cuda_b200.so, which needs the reference's headers"}
    return {k: said[k] for k in built if not built[k]}


def pytest_collection_modifyitems(items):
    missing = reference_missing()
    for item in items:
        needs = NEEDS.get(os.path.basename(str(item.path)), {}).get(getattr(item, "originalname", item.name), ())
        what = [missing[n] for n in needs if n in missing]
        if what:
            item.add_marker(pytest.mark.skip(reason="no reference checkout, and not built: " + ", ".join(what)))


def gpu_available():
    try:
        import qtts_b200 as Q
        return Q.lib().qtb_device_count() > 0
    except Exception:
        return False


@pytest.fixture(scope="session")
def have_gpu():
    if not gpu_available():
        pytest.fail("GPU test selected but no CUDA device / engine library is available")
    return True
