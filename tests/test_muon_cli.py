"""The commands' learning rate of the Muon matrices."""
import argparse

from mx_rcnn_amd.core import launch


def test_default_rate():
    a = launch.add_optimizer_args(argparse.ArgumentParser()).parse_args([])
    assert a.optimizer == 'sgd'
    for lr in (0.001, 0.005):  # the commands' own rates: filters of random-init networks diverge above 0.002
        p = launch.optimizer_params(lr, 0.9, 5e-4, 1000, False, muon_lr_mult=a.muon_lr_mult)
        assert 0.0004 <= p['learning_rate'] * p['muon_lr_mult'] <= 0.002
    b = launch.add_optimizer_args(argparse.ArgumentParser()).parse_args(['--optimizer', 'muon', '--muon-lr-mult', '20'])
    assert (b.optimizer, b.muon_lr_mult) == ('muon', 20.0)
