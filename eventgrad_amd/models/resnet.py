"""CIFAR ResNet family re-implemented from dcifar10/common/resnet.hpp.

Structure (resnet.hpp:111-157): 3x3 stem conv 3->64 (stride 1, no maxpool —
the CIFAR variant), 4 stages at 64/128/256/512 channels with strides
1/2/2/2, avg_pool2d(4), fc. BasicBlock = 2x(3x3 conv + BN), expansion 1
(resnet.hpp:11-54); BottleNeck = 1-3-1 convs, expansion 4 (resnet.hpp:56-109);
1x1-conv+BN downsampler when shape changes; all convs bias-free
(resnet.hpp:3-9).

The reference's ``make_layer`` pushes one block with the stride/downsampler
and then ``blocks`` MORE (resnet.hpp:172-178), so each stage has layers[i]+1
blocks: "ResNet18" = ResNet<BasicBlock>({2,2,2,2}) actually has 12 basic
blocks, 17,444,682 parameters in 86 named tensors. We keep
that behaviour under the ``quirk=True`` models (``resnet18q`` — the
configuration the reference's CIFAR-10 baselines and message counts are
quoted on) and also provide standard counts (``resnet18``).

Every conv is followed by a norm: batch norm, as in the reference, or group
norm (``norm_factory``), which keeps no statistics outside the parameters that
the ranks exchange.
"""

from __future__ import annotations

from torch import nn

from ..ops import functional as O
from .layers import BatchNorm2d, Conv2d, conv_norm


def conv_op(in_ch, out_ch, k, stride, padding):
    # resnet.hpp:3-9 — bias-free conv
    return Conv2d(in_ch, out_ch, k, stride=stride, padding=padding, bias=False)


class Downsampler(nn.Module):
    """1x1 conv + norm shortcut (resnet.hpp:166-171)."""

    def __init__(self, in_ch, out_ch, stride, norm=BatchNorm2d):
        super().__init__()
        self.conv = conv_op(in_ch, out_ch, 1, stride, 0)
        self.bn = norm(out_ch)

    def forward(self, x):
        return conv_norm(self.conv, self.bn, x)


class BasicBlock(nn.Module):
    expansion = 1

    def __init__(self, in_ch, out_ch, stride=1, downsample: bool = False,
                 norm=BatchNorm2d):
        super().__init__()
        self.conv1 = conv_op(in_ch, out_ch, 3, stride, 1)
        self.bn1 = norm(out_ch)
        self.conv2 = conv_op(out_ch, out_ch, 3, 1, 1)
        self.bn2 = norm(out_ch)
        self.downsampler = (Downsampler(in_ch, out_ch * self.expansion, stride,
                                        norm)
                            if downsample else None)

    def forward(self, x):
        if not self.bn1.batch_statistics:
            residual = (self.downsampler(x) if self.downsampler is not None
                        else x)
            out = conv_norm(self.conv1, self.bn1, x, relu=True)
            return self.bn2(self.conv2(out), activation="relu",
                            residual=residual)
        # bn1 -> conv2 is single-consumer: conv2's dgrad epilogue can
        # accumulate bn1's backward stats (ops/functional.py)
        f1 = O.can_fuse_dgrad_stats(self.bn1, self.conv2, x)
        out = self.bn1(self.conv1(x, bn_stats=True), fuse_relu=True,
                       stats_ready=True, stats_consumer=f1)
        # residual FIRST: the downsampler's conv+BN use the same shared
        # per-channel-count stats workspace as the conv2->bn2 pair below —
        # interleaving them corrupts both stats streams
        residual = self.downsampler(x) if self.downsampler is not None else x
        out = self.conv2(out, bn_stats=True,
                         dgrad_stats_bn=self.bn1 if f1 else None)
        # block tail: bn2 -> add+relu with bn2's backward stats fused into
        # the add_relu backward kernel (ops/functional.py::bn_add_relu)
        return O.bn_add_relu(self.bn2, out, residual, stats_ready=True)


class BottleNeck(nn.Module):
    expansion = 4

    def __init__(self, in_ch, out_ch, stride=1, downsample: bool = False,
                 norm=BatchNorm2d):
        super().__init__()
        self.conv1 = conv_op(in_ch, out_ch, 1, 1, 0)
        self.bn1 = norm(out_ch)
        self.conv2 = conv_op(out_ch, out_ch, 3, stride, 1)
        self.bn2 = norm(out_ch)
        self.conv3 = conv_op(out_ch, out_ch * self.expansion, 1, 1, 0)
        self.bn3 = norm(out_ch * self.expansion)
        self.downsampler = (Downsampler(in_ch, out_ch * self.expansion, stride,
                                        norm)
                            if downsample else None)

    def forward(self, x):
        if not self.bn1.batch_statistics:
            residual = (self.downsampler(x) if self.downsampler is not None
                        else x)
            out = conv_norm(self.conv1, self.bn1, x, relu=True)
            out = conv_norm(self.conv2, self.bn2, out, relu=True)
            return self.bn3(self.conv3(out), activation="relu",
                            residual=residual)
        f1 = O.can_fuse_dgrad_stats(self.bn1, self.conv2, x)
        out = self.bn1(self.conv1(x, bn_stats=True), fuse_relu=True,
                       stats_ready=True, stats_consumer=f1)
        f2 = O.can_fuse_dgrad_stats(self.bn2, self.conv3, out)
        out = self.bn2(self.conv2(out, bn_stats=True,
                                  dgrad_stats_bn=self.bn1 if f1 else None),
                       fuse_relu=True, stats_ready=True, stats_consumer=f2)
        residual = self.downsampler(x) if self.downsampler is not None else x
        out = self.conv3(out, bn_stats=True,
                         dgrad_stats_bn=self.bn2 if f2 else None)
        return O.bn_add_relu(self.bn3, out, residual, stats_ready=True)


class CifarResNet(nn.Module):
    """The classic CIFAR-10 ResNet of He et al. (resnet-20/32/44/56...):
    3x3 stem 3->16, three stages at 16/32/64 channels with n blocks each
    (depth = 6n+2), global avg_pool(8), fc. Provided because the
    BASELINE configs name "ResNet-20"; the reference's CODE builds the
    quirk ResNet<BasicBlock>{2,2,2,2} instead — the
    flagship benchmark uses that quirk model for fidelity.
    """

    def __init__(self, n: int, num_classes: int = 10, norm=BatchNorm2d):
        super().__init__()
        self.in_channels = 16
        self.norm = norm
        self.conv = conv_op(3, 16, 3, 1, 1)
        self.bn = norm(16)
        self.layer1 = self._make_stage(16, n, 1)
        self.layer2 = self._make_stage(32, n, 2)
        self.layer3 = self._make_stage(64, n, 2)
        from .layers import Linear
        self.fc = Linear(64, num_classes)

    def _make_stage(self, out_ch, blocks, stride):
        layers = [BasicBlock(self.in_channels, out_ch, stride,
                             downsample=(stride != 1
                                         or self.in_channels != out_ch),
                             norm=self.norm)]
        self.in_channels = out_ch
        for _ in range(blocks - 1):
            layers.append(BasicBlock(out_ch, out_ch, norm=self.norm))
        return nn.Sequential(*layers)

    def forward(self, x):
        x = O.to_compute(x)
        out = conv_norm(self.conv, self.bn, x, relu=True)
        out = self.layer1(out)
        out = self.layer2(out)
        out = self.layer3(out)
        out = O.avg_pool(out, 8)
        out = O.flatten_features(out)
        out = self.fc(out)
        return out if self.training else O.log_softmax(out)


class ResNet(nn.Module):
    def __init__(self, block, layers, num_classes=10, quirk=True,
                 norm=BatchNorm2d):
        super().__init__()
        self.in_channels = 64
        self.norm = norm
        self.conv = conv_op(3, 64, 3, 1, 1)
        self.bn = norm(64)
        self.layer1 = self._make_layer(block, 64, layers[0], 1, quirk)
        self.layer2 = self._make_layer(block, 128, layers[1], 2, quirk)
        self.layer3 = self._make_layer(block, 256, layers[2], 2, quirk)
        self.layer4 = self._make_layer(block, 512, layers[3], 2, quirk)
        from .layers import Linear
        self.fc = Linear(512 * block.expansion, num_classes)

    def _make_layer(self, block, out_ch, blocks, stride, quirk):
        layers = []
        downsample = (stride != 1
                      or self.in_channels != out_ch * block.expansion)
        layers.append(block(self.in_channels, out_ch, stride, downsample,
                            norm=self.norm))
        self.in_channels = out_ch * block.expansion
        # reference quirk (resnet.hpp:172-178): `blocks` MORE blocks after the
        # strided one (layers[i]+1 total); standard builds blocks-1 more.
        extra = blocks if quirk else blocks - 1
        for _ in range(extra):
            layers.append(block(self.in_channels, out_ch, norm=self.norm))
        return nn.Sequential(*layers)

    def forward(self, x):
        x = O.to_compute(x)
        out = conv_norm(self.conv, self.bn, x, relu=True)
        out = self.layer1(out)
        out = self.layer2(out)
        out = self.layer3(out)
        out = self.layer4(out)
        out = O.avg_pool(out, 4)
        out = O.flatten_features(out)
        out = self.fc(out)
        return out if self.training else O.log_softmax(out)


_CONFIGS = {
    "resnet18": (BasicBlock, (2, 2, 2, 2)),
    "resnet34": (BasicBlock, (3, 4, 6, 3)),
    "resnet50": (BottleNeck, (3, 4, 6, 3)),
    "resnet101": (BottleNeck, (3, 4, 23, 3)),
    "resnet152": (BottleNeck, (3, 8, 36, 3)),
}


def resnet_factory(name: str, num_classes: int = 10, norm=BatchNorm2d):
    # classic CIFAR depths: resnet20/32/44/56 (depth = 6n+2)
    if name in ("resnet20", "resnet32", "resnet44", "resnet56"):
        n = (int(name[6:]) - 2) // 6
        return CifarResNet(n, num_classes, norm)
    quirk = name.endswith("q")
    base = name[:-1] if quirk else name
    if base not in _CONFIGS:
        raise ValueError(f"unknown resnet {name!r}")
    block, layers = _CONFIGS[base]
    return ResNet(block, layers, num_classes, quirk=quirk, norm=norm)
