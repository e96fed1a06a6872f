"""The optimizer with 8-bit state under the fault-tolerance harness: a script that uses it is killed and relaunched on
one of two replicas, heals the 8-bit moments from the other, and both then commit identical states."""
import json

from shift_b200.control.session import Session
from test_transparent_cpu import SCRIPT, _ports


def test_8_bit_state_heals_from_a_live_peer(tmp_path):
    text = SCRIPT.read_text()
    assert "torch.optim.AdamW(" in text
    script = tmp_path / "train.py"
    script.write_text("from shift_b200.optim import AdamW\n" + text.replace("torch.optim.AdamW(", "AdamW("))
    lh, mp, sp = _ports(3)
    cfg = {"entry_module": "shift_b200.ft.transparent", "train_args": ["--script", str(script)],
           "lighthouse_port": lh, "master_port": mp, "store_port_base": sp + 1000 if sp < 60000 else 20000,
           "min_replicas": 1, "heartbeat_timeout_ms": 400, "join_timeout_ms": 300, "quorum_tick_ms": 20,
           "target_steps": 100000}
    cpath = tmp_path / "cfg.json"
    cpath.write_text(json.dumps(cfg))
    s = Session(tmp_path, "tr8", cpath, replicas=2, seconds=600)
    s.start(timeout=120)
    try:
        s.await_(lambda: s.last_step(1) >= 5, 120, "step 5")
        rec = s.fault(1, "launcher", timeout=120)
        assert rec["restored_hashes_match"]
        s.await_(lambda: s.last_step(1) >= rec["joint_step"] + 3, 120, "3 joint commits")
    finally:
        s.finish()
    by_step = {}
    for r in s.reader.all_rows:
        if r["kind"] == "commit" and r["step"] > rec["joint_step"] and r["participants"] == 2:
            by_step.setdefault(r["step"], {})[r["rid"]] = r["hashes"]
    joint = [v for v in by_step.values() if len(v) == 2]
    assert joint and all(v[0] == v[1] for v in joint)
