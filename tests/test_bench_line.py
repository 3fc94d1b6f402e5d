"""The line that bench.py prints: short enough that whoever keeps a few kilobytes of output keeps all of it."""
import json

import bench


def record():
    """A run's record at its usual extent: 40 kernels with their tables, in the run itself and in the two further configurations."""
    table = {f'kernel_number_{i}': {'launches_per_step': 1.0, 'ms_per_step': 1.2345678901234567, 'avg_launch_ms': 1.2345678901234567, 'bound': 'mfma',
                                    'achieved': 123.45678901234567, 'unit': 'TFLOP/s', 'frac': 0.12345678901234567} for i in range(40)}
    roof = {'bound': 'mfma', 'kernel': 'lstm_fwd_fused_I2', 'achieved': 120.59119171569336, 'peak': 157.3, 'unit': 'TFLOP/s', 'frac': 0.7666318608753551,
            'traffic': 4860000000.0, 'traffic_unit': 'bytes/launch', 'avg_launch_ms': 3.445841109752655, 'launches': 60,
            'algorithmic_work_per_launch': 415538085888.0, 'all_kernels_ms_per_step': {k: v['ms_per_step'] for k, v in table.items()}, 'note': 'n' * 300}
    one = {'metric': 'm' * 45, 'value': 63123.45678901234, 'unit': 'trajectories/s', 'n_gpus': 1, 'steps': 20, 'warmup': 5, 'ms_per_step': 64.88765432101234,
           'higher_is_better': True, 'scaling': 'weak', 'vs_baseline': None, 'dtype': 'f32', 'data': 'synthetic',
           'config': {'workload': 'w' * 200, 'global_batch': 4096, 'seq_len': 128, 'parallelism': 'dp1'}, 'roofline': roof, 'kernels': table}
    return {**one, 'last_step_metrics': {f'metric_{i}': 0.12345678901234567 for i in range(8)}, 'cpu_baseline': {'value': 66.68, 'sample': 's' * 400},
            'extra_configs': {'config5': dict(one), 'config3': dict(one), 'config9': {'value': None, 'error': 'e' * 100}}}


def test_the_line_is_short_and_keeps_its_contract():
    full = record()
    line = bench.short_line(full)
    assert len(json.dumps(full)) > 15000 and len(json.dumps(line)) < 4000
    for k in ('metric', 'value', 'unit', 'n_gpus', 'steps', 'warmup', 'ms_per_step', 'higher_is_better', 'scaling', 'vs_baseline', 'dtype', 'data', 'config',
              'cpu_baseline'):
        assert line[k] == full[k]
    assert line['roofline']['achieved'] == full['roofline']['achieved'] and 'kernels' in full and 'all_kernels_ms_per_step' in full['roofline']
    for n in ('config3', 'config5'):
        assert line['extra_configs'][n]['value'] == full['extra_configs'][n]['value'] and line['extra_configs'][n]['roofline']['frac']
    assert line['extra_configs']['config9'] == {'value': None, 'error': 'e' * 100}
    assert bench.short_line({'metric': 'm', 'value': 1.0, 'roofline': None}) == {'metric': 'm', 'value': 1.0, 'roofline': None}

