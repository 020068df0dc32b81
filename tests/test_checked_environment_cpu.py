"""Checked mode follows ``os.environ``, whatever object a program puts there."""
import os

import pytest

from arctic_platform_b200.utils import checked


@pytest.mark.parametrize("value,on", [("1", True), ("0", False), ("", False), ("false", False), (None, False)])
def test_checked_mode_follows_another_environment(monkeypatch, value, on):
    monkeypatch.setenv("APB_DEBUG_CHECKS", "0" if on else "1")
    monkeypatch.setattr(os, "environ", {} if value is None else {"APB_DEBUG_CHECKS": value})
    assert checked.enabled() == on
