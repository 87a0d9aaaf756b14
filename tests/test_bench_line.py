"""The benchmark's stdout line: short enough for a reader that keeps the last
3,000 characters, with every key that such a line must have."""
import importlib.util
import json
import os

from conftest import REPO


def test_line_is_short_and_complete():
    spec = importlib.util.spec_from_file_location("bench_module", os.path.join(REPO, "bench.py"))
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    x, text = 1234.5678901234567, "a" * 180
    rows = [{"density": x, "us_per_step": x, "legal_gbs": x}] * 60
    full = {"metric": bench.METRIC, "value": x, "unit": bench.UNIT, "n_gpus": 1, "steps": 20, "warmup": 5,
            "ms_per_step": x, "us_per_step": x, "higher_is_better": True, "scaling": "strong", "vs_baseline": None,
            "dtype": "f16", "data": "synthetic",
            "config": {"workload": text, "mask": text, "batch": 1, "density": 0.01},
            "e2e": {"value": x, "unit": "GB/s", "h2d_bytes_per_step": 35136, "d2h_bytes_per_step": 16,
                    "us_per_step": x, "breakdown": {"what": text, "a": x}, "what": text * 5},
            "gpu_launches": 20, "timing": {"count": 4600, "median_us": x, "what": text},
            "parity": {"support": True, "max_abs_err": x, "method": text}, "roofline": {"frac": x, "source": text},
            "cpu_baseline": {"value": x, "sample": text, "others": {"dense": {"value": x, "sample": text}}},
            "clocks": {"sm_mhz": 1965.0, "sm_max_mhz": 1965, "reasons": []}, "cold": {"us_per_step": x, "what": text}}
    full.update({name: rows for name in bench.SECTIONS})
    line, sections = bench.split_line(full)
    assert len(json.dumps(line)) < 3000
    assert set(full) - set(line) == set(bench.SECTIONS) == set(sections) - {"e2e"}
    assert sections["sweep"] == rows and set(sections["e2e"]) == {"breakdown", "what"}
    assert set(line["e2e"]) == {"value", "unit", "h2d_bytes_per_step", "d2h_bytes_per_step", "us_per_step"}
    assert abs(line["value"] - x) <= 1e-5 * x and line["config"] == full["config"]
