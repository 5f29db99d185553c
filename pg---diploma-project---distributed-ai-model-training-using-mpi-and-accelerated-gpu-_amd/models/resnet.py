"""ResNet-50 (torchvision-identical keys)
("ResNet-50 ImageNet-shape 224x224 synthetic DDP").

Not part of the reference scripts; added because the benchmark plan names it as
the MFMA-conv + all-reduce-bucketing stress configuration.
"""
from typing import List, Optional

import torch
from torch import nn

from ..ops.nn import Conv1x1Ckpt8, GroupNormAct
from .mobilenet_v2 import check_variant


def _conv1(cin: int, cout: int, stride: int, act_ckpt: str) -> nn.Module:
    return Conv1x1Ckpt8(cin, cout, stride) if act_ckpt != "none" else nn.Conv2d(cin, cout, 1, stride, bias=False)


def _norm(c: int, norm: str, act_ckpt: str, act: str = "none") -> nn.Module:
    """BatchNorm2d, or group norm in 32 groups with the activation in the same pass."""
    return GroupNormAct(32, c, act, ckpt8=act_ckpt != "none") if norm == "group" else nn.BatchNorm2d(c)


class Bottleneck(nn.Module):
    expansion = 4

    def __init__(self, inplanes: int, planes: int, stride: int = 1,
                 downsample: Optional[nn.Module] = None, norm: str = "batch", act_ckpt: str = "none"):
        super().__init__()
        self.conv1 = _conv1(inplanes, planes, 1, act_ckpt)
        self.bn1 = _norm(planes, norm, act_ckpt, "relu")
        self.conv2 = nn.Conv2d(planes, planes, 3, stride, 1, bias=False)
        self.bn2 = _norm(planes, norm, act_ckpt, "relu")
        self.conv3 = _conv1(planes, planes * 4, 1, act_ckpt)
        self.bn3 = _norm(planes * 4, norm, act_ckpt)
        self.relu = nn.ReLU(inplace=True)
        self.act = nn.Identity() if norm == "group" else self.relu   # of bn1, bn2
        self.downsample = downsample
        self.stride = stride

    def forward(self, x):
        identity = x
        out = self.act(self.bn1(self.conv1(x)))
        out = self.act(self.bn2(self.conv2(out)))
        out = self.bn3(self.conv3(out))
        if self.downsample is not None:
            identity = self.downsample(x)
        return self.relu(out + identity)


class ResNet(nn.Module):
    def __init__(self, layers: List[int], num_classes: int = 1000, norm: str = "batch", act_ckpt: str = "none"):
        """``norm``, ``act_ckpt``: as MobileNetV2's."""
        super().__init__()
        check_variant(norm, act_ckpt)
        self.norm, self.act_ckpt = norm, act_ckpt
        self.inplanes = 64
        self.conv1 = nn.Conv2d(3, 64, 7, 2, 3, bias=False)
        self.bn1 = _norm(64, norm, act_ckpt, "relu")
        self.relu = nn.Identity() if norm == "group" else nn.ReLU(inplace=True)
        self.maxpool = nn.MaxPool2d(3, 2, 1)
        self.layer1 = self._make_layer(64, layers[0])
        self.layer2 = self._make_layer(128, layers[1], 2)
        self.layer3 = self._make_layer(256, layers[2], 2)
        self.layer4 = self._make_layer(512, layers[3], 2)
        self.avgpool = nn.AdaptiveAvgPool2d((1, 1))
        self.fc = nn.Linear(512 * 4, num_classes)
        for m in self.modules():
            if isinstance(m, nn.Conv2d):
                nn.init.kaiming_normal_(m.weight, mode="fan_out", nonlinearity="relu")
            elif isinstance(m, (nn.BatchNorm2d, GroupNormAct)):
                nn.init.ones_(m.weight)
                nn.init.zeros_(m.bias)

    def _make_layer(self, planes: int, blocks: int, stride: int = 1):
        downsample = None
        if stride != 1 or self.inplanes != planes * 4:
            downsample = nn.Sequential(_conv1(self.inplanes, planes * 4, stride, self.act_ckpt),
                                       _norm(planes * 4, self.norm, self.act_ckpt))
        layers = [Bottleneck(self.inplanes, planes, stride, downsample, self.norm, self.act_ckpt)]
        self.inplanes = planes * 4
        for _ in range(1, blocks):
            layers.append(Bottleneck(self.inplanes, planes, norm=self.norm, act_ckpt=self.act_ckpt))
        return nn.Sequential(*layers)

    def forward(self, x):
        x = self.maxpool(self.relu(self.bn1(self.conv1(x))))
        x = self.layer4(self.layer3(self.layer2(self.layer1(x))))
        return self.fc(torch.flatten(self.avgpool(x), 1))


def resnet50(num_classes: int = 1000, pretrained: Optional[str] = None, **kw) -> ResNet:
    model = ResNet([3, 4, 6, 3], num_classes=num_classes, **kw)
    if pretrained:
        sd = torch.load(pretrained, map_location="cpu", weights_only=True)
        if sd["fc.weight"].shape[0] != num_classes:
            sd = {k: v for k, v in sd.items() if not k.startswith("fc.")}
            missing, unexpected = model.load_state_dict(sd, strict=False)
            # the norms' weights have the same names in both kinds, batch statistics only one has
            if any(k.endswith("running_mean") for k in (*missing, *unexpected)):
                raise ValueError(f"{pretrained} holds another kind of norm than norm={model.norm!r}")
        else:
            model.load_state_dict(sd)
    return model
