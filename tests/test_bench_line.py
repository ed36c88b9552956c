"""The line that bench.py prints: what it has to hold, and short enough to be kept whole by a log's tail."""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _bench():
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    import bench
    return bench


def _entry(**kw):
    x = 0.123456789012345
    return dict(ms=x, frac=x, queries_per_s=x * 1e6, pairs_per_s=x * 1e12, executed_flops=x * 1e14, ms_plain_entry_point=x,
                algorithmic_over_fp32_matrix_peak=x, verified={"verified": True, "recall": 1.0, "queries": 64}, **kw)


def _record():
    """A record with as many entries in each leg as a run with the default arguments makes."""
    x = 0.123456789012345
    fused = dict(_entry(), roofline=_entry(), workload="w" * 200,
                 grid=[_entry(d=d, k=k) for d in (8, 16, 32) for k in (4, 16, 32)],
                 long_lists=[_entry(d=d, k=k) for d in (8, 16, 32) for k in (64, 128, 256)],
                 mfma_f32=dict(_entry(), roofline=_entry()), bf16x3=dict(_entry(), roofline=_entry()),
                 few_queries={"cases": [_entry(d=8, k=k) for k in (32, 64, 256)]})
    gemm = dict(distance_roofline=dict(frac=x, hbm_frac=x), distance_bf16x3=dict(ms=x, roofline=_entry()),
                fused_alternative=dict(ms=x, roofline=_entry()), selection_frac=x, distance_ms=x, selection_ms=x,
                end_to_end_ms=x)
    return {"metric": "m" * 60, "value": 1e12 * x, "unit": "elements/s", "n_gpus": 1, "steps": 20, "warmup": 5,
            "ms_per_step": x, "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "f32",
            "data": "synthetic", "config": {"workload": "c" * 150}, "roofline": _entry(bound="hbm", traffic="t" * 400),
            "verified": {"verified": True}, "calibration": _entry(),
            "sweep": [_entry(k=k, block_size=b, tuned=i == 4) for k in (16, 32, 128, 512, 2048) for b in (128, 256, 512)
                      for i in range(5)],
            "hard_inputs": [_entry(rows=n, k=k, tuned=t) for n in ("ascending", "descending", "256-values")
                            for k in (32, 256) for t in (False, True)],
            "bits_sq": [_entry(rows=n, k=k) for n in (64, 256) for k in (16, 64)], "gemm_knn": gemm, "fused": fused,
            "cpu_baseline": {"value": x, "unit": "elements/s", "sample": "s" * 250, "serial": {"value": x, "sample": "s" * 150}}}


def test_the_line_is_short_and_holds_the_headline():
    bench = _bench()
    record = _record()
    record["summary"] = bench.summarise(record)
    line = json.dumps(bench.line_of(record))
    assert len(json.dumps(record)) > 8000  # what a line of everything would be
    assert len(line) < 6000
    held = json.loads(line)
    for key in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling",
                "vs_baseline", "dtype", "data", "config", "roofline"):
        assert held[key] == record[key]
    assert held["summary"]["all_verified"] is True and held["summary"]["fused_grid_ms"]["d32_k32"] == 0.123


def test_a_run_of_one_leg_has_a_line_too():
    bench = _bench()
    record = {key: None for key in ("metric", "value", "unit")}
    record["summary"] = bench.summarise(record)
    assert set(bench.line_of(record)) == {"metric", "value", "unit", "summary"}
