"""Flags of the factories' presets that the reference does not have."""
import pytest

import derl_amd as derl


@pytest.mark.parametrize("env_id", ["BreakoutNoFrameskip-v4", "Hopper-v2"])
def test_the_optimizer_is_a_flag_of_the_command_line(env_id):
  parse = lambda *argv: derl.get_args(atari_defaults=derl.PPOFactory.get_parser_defaults("atari"),  # noqa: E731
                                      mujoco_defaults=derl.PPOFactory.get_parser_defaults("mujoco"),
                                      args=["--env-id", env_id, *argv], logdir=False, call_log_args=False)
  assert parse().optimizer == "adam"
  assert parse("--optimizer", "muon", "--lr", "1e-3").optimizer == "muon"
  with pytest.raises(SystemExit):
    parse("--optimizer", "sgd")
  assert derl.PPOFactory.get_kwargs("mujoco")["optimizer"] == "adam"
