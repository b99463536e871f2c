"""The package without the extension that Int4Linear and token_logprobs call (another torch, a tree with the library alone): all else is there."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_only_its_operators_raise():
    code = ("import sys, warnings\n"
            "sys.modules['m2_amd._answer_calls'] = None\n"
            "with warnings.catch_warnings(record=True) as seen:\n"
            "    warnings.simplefilter('always')\n"
            "    import m2_amd\n"
            "assert any('_answer_calls' in str(w.message) and 'build' in str(w.message) for w in seen)\n"
            "import torch\n"
            "cfg = m2_amd.m2_bert_80m(128)\n"
            "cfg.num_hidden_layers = 1\n"
            "m2_amd.BertModel(cfg).load_state_dict(m2_amd.seeded_state_dict(cfg, 1))\n"
            "lin = m2_amd.Int4Linear.from_weight(torch.ones(4, 32), None, 32)\n"
            "assert (lin.dequantized() - 1).abs().max() < 0.01\n"
            "for call in (lambda: lin(torch.ones(1, 32)), lambda: m2_amd.token_logprobs(torch.ones(1, 32))):\n"
            "    try:\n"
            "        call()\n"
            "    except RuntimeError as e:\n"
            "        assert 'build' in str(e)\n"
            "    else:\n"
            "        raise AssertionError\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
