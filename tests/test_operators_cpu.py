"""CPU tests of the operators beside the per-bucket op: what they refuse, before
any device is touched, and the sizes they report."""
from __future__ import annotations

import pytest
import torch


def test_scan_shapes_and_workspaces(race):
    from race_attention_kernel_amd import abi

    ok = abi.scan_shape(8, 4096, 2048)
    st, nbytes, floats = abi.gated_scan_workspace_bytes(ok)
    assert st == abi.RACE_SUCCESS and nbytes == 0 and floats == 8 * 32 * 2048  # 128-token tiles
    assert abi.gated_scan_workspace_bytes(abi.scan_shape(32, 4096, 2048))[2] == 32 * 128 * 2048  # 32-token tiles
    # Few channels: the tokens are split, and the pairs of the segments need room.
    st, nbytes, _ = abi.gated_scan_workspace_bytes(abi.scan_shape(8, 65536, 64))
    assert st == abi.RACE_SUCCESS and nbytes > 0
    st, back, _ = abi.gated_scan_workspace_bytes(abi.scan_shape(8, 65536, 64), backward=True)
    assert st == abi.RACE_SUCCESS and 0 < back <= nbytes
    st, nbytes, floats = abi.gated_scan_workspace_bytes(abi.scan_shape(0, 5, 64))
    assert (st, nbytes, floats) == (abi.RACE_SUCCESS, 0, 0)
    for bad in (abi.scan_shape(65536, 1, 4), abi.scan_shape(-1, 1, 4), abi.scan_shape(1, -1, 4),
                abi.scan_shape(1, 2 ** 31 - 1, 4), abi.scan_shape(1, 1, 0), abi.scan_shape(1, 1, 65537),
                abi.scan_shape(1, 1, 4, dtype=2), abi.scan_shape(1, 1, 4, gate_form=2),
                abi.scan_shape(1, 1, 4, lengths_group=0),
                abi.RaceScanShape(1, 9, 4, 0, (1 << 20) + 1, 0, 4, 0, 0, 1, 1),
                abi.RaceScanShape(1, 9, 4, -4, 4, 0, 4, 0, 0, 1, 1)):
        assert abi.gated_scan_workspace_bytes(bad)[0] == abi.RACE_ERROR_INVALID_VALUE


def test_scan_refuses_bad_pointers_on_the_host(race):
    from race_attention_kernel_amd import abi

    sh = abi.scan_shape(2, 300, 64)
    bad = abi.RACE_ERROR_INVALID_VALUE
    assert abi.gated_scan_fwd(0, 16, None, None, 16, None, None, sh, None, 0, 0) == bad
    assert abi.gated_scan_fwd(8, 16, None, None, 16, None, None, sh, None, 0, 0) == bad
    assert abi.gated_scan_fwd(16, 16, 4, None, 16, None, None, sh, None, 0, 0) == bad
    assert abi.gated_scan_bwd(16, 16, None, 16, None, None, 16, None, None, sh, None, 0, 0) == bad
    assert abi.gated_scan_bwd(16, 16, None, 8, None, 16, 16, None, None, sh, None, 0, 0) == bad
    split = abi.scan_shape(8, 65536, 64)  # needs a workspace
    assert abi.gated_scan_fwd(16, 16, None, None, 16, None, None, split, None, 0, 0) == bad
    # Nothing to do touches no device.
    assert abi.gated_scan_fwd(0, 0, None, None, 0, None, None, abi.scan_shape(0, 5, 64), None, 0, 0) == 0
    assert abi.gated_scan_bwd(0, 0, None, 0, None, 0, None, None, None, sh, None, 0, 0) == 0


def test_scan_binding_validates_inputs_on_the_host(race):
    x = torch.randn(2, 5, 8)
    with pytest.raises(RuntimeError, match="race_gated_scan: x lives on the CPU"):
        race.race_gated_scan(x, x)
    with pytest.raises(RuntimeError, match="x lives on the CPU"):
        race.race_gated_scan_carry(x, x, torch.zeros(2, 8))
    with pytest.raises(ValueError, match="gate_form"):
        race.race_gated_scan(x, x, gate_form="tanh")


def test_norm_rope_refuses_on_the_host(race):
    from race_attention_kernel_amd import abi

    bad = abi.RACE_ERROR_INVALID_VALUE
    ok = abi.norm_rope_shape(2, 300, 12, 4, 64, 32)
    st, nbytes = abi.norm_rope_bwd_workspace_bytes(ok)
    assert st == abi.RACE_SUCCESS and nbytes == 1536 * 64 * 4
    assert abi.norm_rope_bwd_workspace_bytes(abi.norm_rope_shape(1 << 15, 1 << 15, 1, 0, 64, 32))[0] == abi.RACE_SUCCESS
    assert abi.norm_rope_bwd_workspace_bytes(abi.norm_rope_shape(1 << 15, (1 << 15) + 1, 1, 0, 64, 32))[0] == bad
    for kw in (dict(B=-1), dict(T=-1), dict(B=1 << 16, T=1 << 15), dict(Hq=0), dict(Hk=-1), dict(d=0, pairs=0),
               dict(d=257), dict(pairs=33), dict(pairs=-1), dict(sections=[16, 15]), dict(sections=[33, -1]),
               dict(pos_bits=16), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=2), dict(weight_dtype=3)):
        args = dict(B=2, T=300, Hq=12, Hk=4, d=64, pairs=32) | kw
        assert abi.norm_rope_bwd_workspace_bytes(abi.norm_rope_shape(**args))[0] == bad, kw
    assert abi.norm_rope_fwd(0, 16, 16, 16, None, None, 16, 16, ok, 0) == bad
    assert abi.norm_rope_fwd(16, 16, None, 16, None, None, 16, 16, ok, 0) == bad
    assert abi.norm_rope_fwd(16, 16, 16, 16, 4, None, 16, 16, ok, 0) == bad
    assert abi.norm_rope_fwd(16, None, 16, 16, None, None, 16, None, ok, 0) == bad
    assert abi.norm_rope_bwd(16, 16, 16, 16, None, None, 16, 16, 16, 16, 16, None, ok, None, 0, 0) == bad
    # Nothing to do touches no device.
    assert abi.norm_rope_fwd(0, None, None, None, None, None, 0, None, abi.norm_rope_shape(0, 5, 1, 0, 64, 32), 0) == 0
    assert abi.norm_rope_bwd(16, 16, 16, 16, None, None, None, None, 16, 16, None, None, ok, None, 0, 0) == 0
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(RuntimeError, match="race_norm_rope: q lives on the CPU"):
        race.race_norm_rope(x, x)


def test_cross_refuses_on_the_host(race):
    from race_attention_kernel_amd import abi

    bad = abi.RACE_ERROR_INVALID_VALUE
    ok = abi.cross_shape(8, 40, 300, 4, 16, 64)
    for backward in (False, True):
        st, nbytes = abi.cross_workspace_bytes(ok, backward)
        assert st == abi.RACE_SUCCESS and nbytes >= 8 * 64 * 65 * 4
        assert abi.cross_workspace_bytes(abi.cross_shape(0, 40, 300, 4, 16, 64), backward) == (abi.RACE_SUCCESS, 0)
        for args in ((65536, 1, 1, 4, 16, 64), (1, -1, 1, 4, 16, 64), (1, 1, -1, 4, 16, 64), (1, 2 ** 31 - 1, 1, 4, 16, 64),
                     (1, 1, 1, 0, 16, 64), (1, 1, 1, 4, 65, 64), (1, 1, 1, 4, 16, 129), (1, 1, 1, 4, 16, 64, 2),
                     (1, 1, 1, 4, 16, 64, 0, 0)):
            assert abi.cross_workspace_bytes(abi.cross_shape(*args), backward)[0] == bad, args
    assert abi.cross_fwd(None, 16, 16, None, 16, None, ok, 16, 1 << 30, 0) == bad
    assert abi.cross_fwd(16, 16, 16, None, 16, None, ok, 16, 64, 0) == bad
    assert abi.cross_fwd(16, 16, 8, None, 16, None, ok, 16, 1 << 30, 0) == bad
    assert abi.cross_query(16, 4, 16, ok, 0) == bad
    assert abi.cross_bwd(16, 16, 16, None, 16, None, 16, 16, 16, ok, 16, 1 << 30, 0) == bad
    assert abi.cross_bwd(16, 16, 16, None, 16, 16, 16, 16, 16, ok, None, 0, 0) == bad
    # Nothing to do touches no device.
    assert abi.cross_fwd(None, 16, 16, None, None, None, ok, None, 0, 0) == 0
    assert abi.cross_bwd(16, 16, 16, None, 16, 16, None, None, None, ok, None, 0, 0) == 0
    x = torch.zeros(2, 3, 16)
    with pytest.raises(RuntimeError, match="race_cross_fwd: probsQ lives on the CPU"):
        race.race_cross_fwd(x, x, x)
    with pytest.raises(RuntimeError, match="race_cross_state: probsK lives on the CPU"):
        race.race_cross_state(x, x)


def test_frequencies_first_made_under_inference_mode_serve_training(race):
    # An inference tensor could not be saved for a later backward.
    module = race.BatchedACE(64, 4, 4, 1, rope_pairs=16)
    with torch.inference_mode():
        first = module.inv_freq(torch.device("cpu"))
    assert not first.is_inference() and not module.inv_freq(torch.device("cpu")).is_inference()
    leaf = torch.ones(16, requires_grad=True)
    (leaf * module.inv_freq(torch.device("cpu"))).sum().backward()  # saves them
    assert torch.equal(leaf.grad, race.BatchedACE(64, 4, 4, 1, rope_pairs=16).inv_freq(torch.device("cpu")))


def test_modules_pickled_before_the_norm_and_rotation_load(race):
    import pickle

    rows = torch.randn(1, 2, 5, 3, 64)
    for causal in (True, False):
        module = race.BatchedACE(64, 4, 4, 1, causal=causal)
        for name in ("norm_eps", "q_norm", "k_norm", "rope_pairs", "rope_theta", "rope_sections", "rope_interleaved",
                     "_inv_freq"):
            del module.__dict__[name]
        old = pickle.loads(pickle.dumps(module))
        assert torch.equal(old.planes_T, module.planes_T) and old.inv_freq(rows.device) is None
        with pytest.raises(RuntimeError, match="CPU"):  # as far as any module comes here
            old(rows, rows, rows)


def test_copies_and_pickles_make_their_own_frequencies(race):
    import copy
    import pickle

    module = race.CrossACE(64, 4, 4, 1, qk_norm=True, rope_pairs=16, rope_sections=[8, 8], rope_interleaved=True)
    freq = module.inv_freq(torch.device("cpu"))
    for other in (copy.deepcopy(module), copy.copy(module), pickle.loads(pickle.dumps(module))):
        assert not other._inv_freq and torch.equal(other.inv_freq(torch.device("cpu")), freq)
        assert other.rope_sections == [8, 8] and other.rope_interleaved and other.norm_eps == module.norm_eps
        assert sorted(n for n, _ in other.named_parameters()) == ["k_norm", "q_norm"]
    assert module.inv_freq(torch.device("cpu")) is freq


def test_a_decode_step_of_a_rotating_module_needs_its_positions(race):
    # Counted from 0 every step would be rotated as the first.
    Q, state = torch.randn(1, 2, 1, 3, 64), torch.zeros(6, 64 * 64 + 64)
    with pytest.raises(ValueError, match="q_positions are needed"):
        race.CrossACE(64, 4, 4, 1, rope_pairs=16).query(Q, state)
    for options, positions in ((dict(rope_pairs=16), torch.tensor([7])), (dict(), None), (dict(qk_norm=True), None)):
        with pytest.raises(RuntimeError, match="lives on the CPU"):  # past that check
            race.CrossACE(64, 4, 4, 1, **options).query(Q, state, positions)


# (N, T, D, dtype, tokens of a backward tile, segments): the launch shapes of training
# steps, which tests/test_gpu_gated_scan.py runs at these sizes.
SCAN_FORMS = [(105, 1700, 128, 0, 128, 1), (24, 600, 520, 0, 128, 1), (24, 600, 520, 1, 128, 1), (210, 1700, 128, 1, 32, 1),
              (2, 1500, 260, 0, 32, 24), (39, 640, 260, 1, 128, 1), (32, 640, 260, 1, 32, 5), (2, 45000, 256, 0, 32, 118), (8, 65536, 64, 1, 64, 64),
              (8, 4096, 2048, 1, 128, 1), (24, 1531, 520, 0, 128, 1), (32, 4096, 2048, 1, 32, 1), (8, 4096, 1536, 1, 128, 1),
              (24, 1531, 448, 0, 128, 1), (8, 4096, 1280, 1, 32, 6)]


@pytest.mark.parametrize("N, T, D, dtype, tile, segments", SCAN_FORMS)
def test_scan_forms(race, N, T, D, dtype, tile, segments):
    from race_attention_kernel_amd import abi

    sh = abi.scan_shape(N, T, D, dtype=dtype)
    st, back, records = abi.gated_scan_workspace_bytes(sh, backward=True)
    assert st == abi.RACE_SUCCESS and records == N * -(-T // tile) * D
    pairs = N * segments * 2 * D
    assert back == (0 if segments == 1 else 4 * (-(-pairs // 64) * 64))
