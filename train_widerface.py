#!/usr/bin/env python
"""End-to-end face detection training on a .lst dataset such as WIDER FACE (reference
`train_widerface.py`): ResNet when 'resnet' is in --pretrained (or --network), else VGG16."""
import argparse
import logging

from mx_rcnn_amd.config import config
from mx_rcnn_amd.core import launch
from mx_rcnn_amd.core.callback import Speedometer
from mx_rcnn_amd.core.metric import e2e_metrics
from mx_rcnn_amd.core.module import MutableModule
from mx_rcnn_amd.data.load_data import load_gt_roidb_from_list
from mx_rcnn_amd.data.loader import AnchorLoader
from mx_rcnn_amd.parallel import dist as pdist
from mx_rcnn_amd.utils.load_model import do_checkpoint

DEFAULT_NETWORK = 'resnet50'


def init_config():
    """train_widerface.py:20-36"""
    config.TRAIN.BG_THRESH_HI = 0.5
    config.TRAIN.BG_THRESH_LO = 0.0
    config.SCALES = (640,)
    config.MAX_SIZE = 1024
    config.TRAIN.RPN_MIN_SIZE = 10
    config.TRAIN.HAS_RPN = True
    config.END2END = 1
    config.TRAIN.BBOX_NORMALIZATION_PRECOMPUTED = True


def main(args, default_network=DEFAULT_NETWORK):
    rank, world, device = launch.init_runtime(args)
    logging.info('########## TRAIN FASTER-RCNN WITH APPROXIMATE JOINT END2END #############')
    init_config()
    network = args.network if args.network != 'vgg16' or 'resnet' in args.pretrained else 'vgg16'
    if 'resnet' in args.pretrained and network == 'vgg16':
        network = default_network
    model, arg_params, aux_params = launch.build_model(network, args.num_classes, args.pretrained, args.load_epoch,
                                                       args.resume, bn_mom=args.bn_mom)
    if args.synthetic:
        imdb, roidb = launch.synthetic_roidb(args, args.num_classes, flip=not args.no_flip)
    else:
        imdb, roidb = load_gt_roidb_from_list(args.dataset_name, args.lst, args.dataset_root, args.outdata_path,
                                              flip=not args.no_flip)
    fam = launch.family(network)
    train_data = AnchorLoader(model, roidb, batch_size=args.ims_per_gpu, shuffle=not args.no_shuffle,
                              anchor_scales=model.anchor_scales, rank=rank, world_size=world, seed=args.seed,
                              need_mean=args.need_mean, max_gt=1200, raw_images=launch.raw_images(device))
    launch.calibrate_if_random(model, train_data, arg_params)
    mod = MutableModule(model, data_names=['data', 'im_info'], label_names=['gt_boxes'], context=device,
                        fixed_param_prefix=launch.FIXED_PREFIX[fam] if fam == 'resnet' else
                        ['conv1', 'conv2', 'conv3'], mode='e2e', use_graph=not args.eager)
    mod.fit(train_data, eval_metric=e2e_metrics(), epoch_end_callback=do_checkpoint(args.prefix),
            batch_end_callback=Speedometer(args.ims_per_gpu * world, frequent=args.frequent),
            optimizer=args.optimizer,
            optimizer_params=launch.optimizer_params(args.lr, args.mom, args.wd, args.factor_step, args.resume,
                                                     warmup=False, muon_lr_mult=args.muon_lr_mult),
            arg_params=arg_params, aux_params=aux_params, begin_epoch=args.load_epoch, num_epoch=args.num_epoch,
            max_steps=args.max_steps)
    pdist.destroy()
    return mod


def parse_args(argv=None, default_network=DEFAULT_NETWORK):
    p = argparse.ArgumentParser(description='Train Faster R-CNN on a detection list (WIDER FACE)')
    p.add_argument('--dataset-name', dest='dataset_name', default='wider_face')
    p.add_argument('--lst', default='data/trainval.lst')
    p.add_argument('--num-classes', dest='num_classes', type=int, default=2)
    p.add_argument('--outdata-path', dest='outdata_path', default='data')
    p.add_argument('--dataset-root', dest='dataset_root', default='data/WIDER')
    p.add_argument('--pretrained', default='model/%s' % default_network.replace('resnet', 'resnet-'))
    p.add_argument('--load-epoch', dest='load_epoch', type=int, default=0)
    p.add_argument('--prefix', default='model/%s-face' % default_network)
    p.add_argument('--gpus', dest='gpu_ids', default='0')
    p.add_argument('--num_epoch', type=int, default=10)
    p.add_argument('--frequent', type=int, default=20)
    p.add_argument('--kv-store', dest='kv_store', default='device')
    p.add_argument('--need-mean', dest='need_mean', action='store_true')
    p.add_argument('--no-flip', dest='no_flip', action='store_true')
    p.add_argument('--no-shuffle', dest='no_shuffle', action='store_true')
    p.add_argument('--lr', type=float, default=0.001)
    p.add_argument('--mom', type=float, default=0.9)
    p.add_argument('--bn-mom', dest='bn_mom', type=float, default=0.99)
    p.add_argument('--wd', type=float, default=0.0005)
    p.add_argument('--resume', action='store_true')
    p.add_argument('--factor-step', dest='factor_step', type=int, default=50000)
    launch.add_optimizer_args(p)
    launch.add_common_args(p)
    a = p.parse_args(argv)
    if a.network == 'vgg16' and 'resnet' in a.pretrained:
        a.network = default_network
    return a


if __name__ == '__main__':
    main(parse_args())
