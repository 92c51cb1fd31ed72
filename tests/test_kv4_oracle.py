"""Pins of ``oracle/kv4_oracle.py`` and of the torch forms of the 4-bit format, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4_oracle, kv_oracle
from simpler_amd import workloads
from tests.int4_cases import make_int4_case


@pytest.mark.parametrize("group", [32, 64, 128])
def test_evenly_spaced_and_constant_groups_are_exact(group):
    codes = np.random.default_rng(1).integers(0, 16, (5, 256))
    codes[:, ::group], codes[:, 1::group] = 0, 15
    rows = (codes * 0.25 - 1.5).astype(np.float32)
    rows[2] = 3.140625  # constant: scale 0
    got, s, z = kv4_oracle.quantise(rows, group)
    np.testing.assert_array_equal(kv4_oracle.dequantise(got, s, z), rows)
    assert (s[2] == 0).all() and (got[2] == 0).all() and (s[0] == 0.25).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_element_is_off_by_half_a_step_at_most(dtype):
    rows = (torch.randn((7, 3, 128), generator=torch.Generator().manual_seed(2)) * 3).to(dtype)
    codes, s, z = kv4_oracle.quantise(rows.float().numpy(), 64)
    got = kv4_oracle.dequantise(codes, s, z)
    # half a step, and fp16's rounding of the least value (2^-11) and of the step (15 of them)
    bound = s.astype(np.float64) * (0.5 + 15 * 2.0**-11) + np.abs(z.astype(np.float64)) * 2.0**-11
    assert (np.abs(got - rows.double().numpy()).reshape(7, 3, 2, 64) <= bound[..., None]).all()
    torch_codes, ts, tz = workloads.quantize_kv4(rows, 64)
    np.testing.assert_array_equal(torch_codes.numpy(), codes)
    np.testing.assert_array_equal(ts.numpy(), s)
    np.testing.assert_array_equal(tz.numpy(), z)
    np.testing.assert_array_equal(workloads.dequantize_kv4(torch_codes, ts, tz).numpy(), got)


def test_ties_infinities_and_saturation():
    row = np.zeros((1, 32), np.float32)
    row[0, :6] = [0.5, 1.5, 2.5, 15.0, 14.5, 13.5]  # step 1 from 0: halves go to even codes
    codes, s, z = kv4_oracle.quantise(row, 32)
    assert s[0, 0] == 1 and z[0, 0] == 0
    assert codes[0, :6].tolist() == [0, 2, 2, 15, 14, 14]
    row[0, 7] = np.inf
    _, s, z = kv4_oracle.quantise(row, 32)
    assert np.isnan(s[0, 0]) and np.isnan(z[0, 0])
    row[0, 7], row[0, 8] = -3e38, 3e38
    codes, s, z = kv4_oracle.quantise(row, 32)
    assert s[0, 0] == 65504 and z[0, 0] == -65504 and codes[0, 7] == 0 and codes[0, 8] == 15


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("value", [False, True])
def test_every_nibble_of_a_page_holds_one_element(dim, value):
    index = kv4_oracle.nibble_index(16, dim, value)
    assert sorted(index.ravel().tolist()) == list(range(16 * dim))
    codes = torch.randint(0, 16, (2, 3, 16, dim), dtype=torch.uint8, generator=torch.Generator().manual_seed(dim))
    pages = workloads.pack_kv4_pages(codes, value)
    ones = np.zeros((2, 3, 1, 16, 2), np.float16)
    ones[..., 0] = 1
    np.testing.assert_array_equal(kv4_oracle.pages_to_rows(pages.numpy(), ones, value), codes.numpy())


def test_attention_over_one_token_is_its_value_row_and_over_none_zero():
    case = make_int4_case([1, 0, 33], dim=64, group=32, block=16, seed=4)
    out = case.reference()
    v = kv4_oracle.pages_to_rows(case.value_cache.numpy(), case.v_scale.numpy(), True)
    np.testing.assert_allclose(out[0], np.repeat(v[case.block_table[0, 0], :, 0], 4, axis=0), rtol=1e-15)
    assert (out[1] == 0).all()


def test_one_axis_is_the_plain_rope():
    rng = np.random.default_rng(5)
    cos, sin = (t.numpy() for t in workloads.rope_tables(50, 64))
    x, pos = rng.standard_normal((9, 3, 64)).astype(np.float32), rng.integers(0, 50, 9)
    got = kv4_oracle.mrope(x, np.stack([pos, pos * 0, pos * 0 + 7]), [32, 0, 0], cos, sin, False)
    lo, hi = x[..., :32].astype(np.float64), x[..., 32:].astype(np.float64)
    c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
    np.testing.assert_allclose(got, np.concatenate([lo * c[..., :32] - hi * s[..., :32],
                                                    hi * c[..., 32:] + lo * s[..., 32:]], -1), rtol=1e-15, atol=1e-15)
    # three axes with equal positions are one axis, in both orders of the pairs
    for order in (False, True):
        same = kv4_oracle.mrope(x, np.stack([pos] * 3), [12, 10, 10], cos, sin, order)
        np.testing.assert_array_equal(same, got)


def test_slots_are_those_of_the_table():
    rng = np.random.default_rng(6)
    new, lens = np.array([1, 0, 37, 5]), np.array([16, 9, 0, 31])
    table = np.full((4, 5), -1)
    table[0, 0], table[1, 0], table[3, :2] = 11, 12, [13, 14]
    free = rng.permutation(10)
    slots, pos, req, starts, out_lens, granted, left, table2 = kv4_oracle.assign_slots(new, lens, table, free, 10, 16, 50)
    assert left == 10 - 1 - 3 - 1 and starts.tolist() == [0, 1, 1, 38, 43] and granted.tolist() == new.tolist()
    assert table2[0, 1] == free[9] and table2[2, :3].tolist() == free[[8, 7, 6]].tolist() and table2[3, 2] == free[5]
    for b in range(4):
        want = kv_oracle.new_token_slots(table2[b:b + 1], out_lens[b:b + 1], 16, int(new[b]))[0]
        np.testing.assert_array_equal(slots[starts[b]:starts[b + 1]], want)
    assert (slots[43:] == -1).all() and (req[43:] == -1).all() and pos[42] == 35
